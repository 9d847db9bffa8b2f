// Attention over prompts (prompt_attention.cu): what the rest of the library calls.
#pragma once

namespace grinqh {

unsigned take_prompt_timeouts();  // reads and clears the kernel's count of waits that gave up

}  // namespace grinqh
