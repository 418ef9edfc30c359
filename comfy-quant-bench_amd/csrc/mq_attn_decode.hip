// Attention of one new token per sequence over a paged key-value cache: the kernels of mq_attn_decode_kernel.h for
// sequences that are read one by one.
#include "mq_attn_decode_kernel.h"

namespace mq {

int64_t attn_decode_workspace_bytes(int Hq, int H, int D) {
    const int group = Hq / H, rows = group < 16 ? group : 16;
    return 2 * static_cast<int64_t>(decode_groups()) * rows * (D + 2) * 4;
}

int launch_attn_decode(const AttnArgs& a, hipStream_t stream) { return decode<false>(a, stream); }

int64_t attn_decode_counters(int Hq, int H, int64_t B) { return B * H * ((Hq / H + 15) / 16); }

}  // namespace mq
