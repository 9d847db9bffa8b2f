// Attention over the 4-bit cache (kv4_attention.cu): what the rest of the library calls.
#pragma once

namespace grinqh {

unsigned take_kv4_timeouts();  // reads and clears the kernel's count of waits that gave up

}  // namespace grinqh
