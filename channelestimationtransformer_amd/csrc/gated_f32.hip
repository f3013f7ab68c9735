// The gated projection: the matrix products for float tensors.
#include "gated.h"

namespace cet {
namespace gated {

int run_f32(const Args& a, int step, int tile, hipStream_t s) { return run<float>(a, step, tile, s); }

}  // namespace gated
}  // namespace cet
