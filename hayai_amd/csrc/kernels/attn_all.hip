// Translation unit of the attention operators' gfx950 code object, apart from all.hip's so that the two
// compile at the same time.
#include "rope.hip"
#include "kv_pages.hip"
#include "attn_prompt.hip"
#include "attn_decode.hip"
