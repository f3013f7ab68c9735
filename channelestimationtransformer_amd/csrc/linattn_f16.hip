// Linear attention: the chunk kernels for _Float16 tensors.
#include "linattn.h"

namespace cet {
namespace la {

void launch_f16(const Passes& p, bool out, unsigned blocks, hipStream_t s) {
  if (out)
    launch<_Float16, true>(p, blocks, s);
  else
    launch<_Float16, false>(p, blocks, s);
}

}  // namespace la
}  // namespace cet
