// The gated projection: the matrix products for __bf16 tensors.
#include "gated.h"

namespace cet {
namespace gated {

int run_bf16(const Args& a, int step, int tile, hipStream_t s) { return run<__bf16>(a, step, tile, s); }

}  // namespace gated
}  // namespace cet
