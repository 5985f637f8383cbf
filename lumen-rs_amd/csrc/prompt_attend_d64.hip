// Attention of packed sequences, head dim 64.
#include "prompt_attend.hpp"

namespace tqkv {
namespace prompt {
template void launch_prompt<64>(const Args&, Source, hipStream_t);
}  // namespace prompt
}  // namespace tqkv
