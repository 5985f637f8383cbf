// Attention of packed sequences with few rows, head dim 512.
#include "prompt_few.hpp"

namespace tqkv {
namespace prompt {
template void launch_few<512>(const Args&, Source, hipStream_t);
}  // namespace prompt
}  // namespace tqkv
