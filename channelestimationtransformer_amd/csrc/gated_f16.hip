// The gated projection: the matrix products for _Float16 tensors.
#include "gated.h"

namespace cet {
namespace gated {

int run_f16(const Args& a, int step, int tile, hipStream_t s) { return run<_Float16>(a, step, tile, s); }

}  // namespace gated
}  // namespace cet
