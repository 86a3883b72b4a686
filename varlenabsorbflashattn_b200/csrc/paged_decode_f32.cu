// Paged decode attention: the kernels of one type.
#include "paged_decode.cuh"

namespace vafa {
namespace paged {
Plan plan_f32(int D, int R) { return plan_by_dim<float>(D, R); }
}  // namespace paged
}  // namespace vafa
