// Linear attention: the chunk kernels for float tensors.
#include "linattn.h"

namespace cet {
namespace la {

void launch_f32(const Args& a, bool out, unsigned blocks, hipStream_t s) {
  if (out)
    launch<float, true>(a, blocks, s);
  else
    launch<float, false>(a, blocks, s);
}

}  // namespace la
}  // namespace cet
