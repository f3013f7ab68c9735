// Linear attention: the chunk kernels for __bf16 tensors.
#include "linattn.h"

namespace cet {
namespace la {

void launch_bf16(const Passes& p, bool out, unsigned blocks, hipStream_t s) {
  if (out)
    launch<__bf16, true>(p, blocks, s);
  else
    launch<__bf16, false>(p, blocks, s);
}

}  // namespace la
}  // namespace cet
