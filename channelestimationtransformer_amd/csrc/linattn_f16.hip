// Linear attention: the chunk kernels for _Float16 tensors.
#include "linattn.h"

namespace cet {
namespace la {

void launch_f16(const Args& a, bool out, unsigned blocks, hipStream_t s) {
  if (out)
    launch<_Float16, true>(a, blocks, s);
  else
    launch<_Float16, false>(a, blocks, s);
}

}  // namespace la
}  // namespace cet
