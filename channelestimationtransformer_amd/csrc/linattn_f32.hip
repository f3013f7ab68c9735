// Linear attention: the chunk kernels for float tensors.
#include "linattn.h"

namespace cet {
namespace la {

void launch_f32(const Passes& p, bool out, unsigned blocks, hipStream_t s) {
  if (out)
    launch<float, true>(p, blocks, s);
  else
    launch<float, false>(p, blocks, s);
}

}  // namespace la
}  // namespace cet
