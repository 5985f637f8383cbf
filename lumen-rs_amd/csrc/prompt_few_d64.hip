// Attention of packed sequences with few rows, head dim 64.
#include "prompt_few.hpp"

namespace tqkv {
namespace prompt {
template void launch_few<64>(const Args&, Source, hipStream_t);
}  // namespace prompt
}  // namespace tqkv
