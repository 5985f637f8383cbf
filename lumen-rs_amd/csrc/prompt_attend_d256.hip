// Attention of packed sequences, head dim 256.
#include "prompt_attend.hpp"

namespace tqkv {
namespace prompt {
template void launch_prompt<256>(const Args&, Source, hipStream_t);
}  // namespace prompt
}  // namespace tqkv
