// Paged decode attention, affine layouts of head dim 512.
#include "paged_decode.hpp"

namespace tqkv {
namespace paged {
template int launch_affine<512>(const DecodeArgs&, int, int, int, dim3, hipStream_t, bool);
}  // namespace paged
}  // namespace tqkv
