// Paged decode attention: the kernels of one type.
#include "paged_decode.cuh"

namespace vafa {
namespace paged {
Plan plan_bf16(int D, int R) { return plan_by_dim<__nv_bfloat16>(D, R); }
}  // namespace paged
}  // namespace vafa
