// Attention of prompts in bf16 (prompt_impl.hpp).
#include "prompt_impl.hpp"

namespace dmx {
template hipError_t prompt_launch_typed<false>(const PromptArgs&, const PromptPlan&, hipStream_t);
}
