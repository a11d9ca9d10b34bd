// Attention of prompts in f32 (prompt_impl.hpp).
#include "prompt_impl.hpp"

namespace dmx {
template hipError_t prompt_launch_typed<true>(const PromptArgs&, const PromptPlan&, hipStream_t);
}
