// Attention of packed sequences, head dim 128.
#include "prompt_attend.hpp"

namespace tqkv {
namespace prompt {
template void launch_prompt<128>(const Args&, Source, hipStream_t);
}  // namespace prompt
}  // namespace tqkv
