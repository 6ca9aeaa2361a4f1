// kv_attend.h -- the attention kernels' arguments and launchers (kv_attend.cu chooses).
#pragma once
#include "kv_impl.h"

namespace rmoe {

struct AttendArg {
    Rows q, out;
    const int32_t *table, *lens, *cu;
    float* lse;
    int R, max_blocks, T;
    int group;           // query heads per kv head
    uint32_t group_inv;  // ceil(2^32 / group): x / group = mulhi(x, group_inv) for x < 2^16; 0 for group 1
    float scale;
    int window;
    bool prompts;  // the prompt kernel runs too and takes the requests of more than split_max_rows rows
};

// Adds a workspace to the cache, its counts zeroed when this returns.
cudaError_t add_split_slot(rmoe_kv* kv);

// Rows of a request: its new tokens x the query heads that share a kv head.
static constexpr int PROMPT_MIN_ROWS = 64, PROMPT_PAIR_ROWS = 256, PROMPT_MIN_CTAS = 24;

#ifdef __CUDACC__
// The first key that the query at position p sees (p may be negative, the window up to 2^31 - 1).
__device__ __forceinline__ int first_seen(int window, int p) { return window && p >= window ? p - window + 1 : 0; }

// The most rows of a request that the split kernel takes when the prompt kernel runs too.  The
// prompt kernel works on 256 rows per CTA at several times the split kernel's rate (2048 tokens: 4 to 5
// times, 8192: 4 to 7), but does not split the keys: with few CTAs the split kernel, which always fills
// the chip, is the faster one.  Prompt / split in us (B200, 32 heads over 4, 128 wide, bf16):
//   16 CTAs: 128 tokens 19.8 / 10.9, 128 more on a cache of 8192 152.7 / 127.2
//   24 CTAs: 192 tokens 21.1 / 20.4, 192 more on a cache of 8192 152.0 / 181.2
// 64 wide and f32 cross between 12 and 24 too; f32, 128 wide, 16 CTAs on 8192 loses by the rule (138 / 178).
// Called by every thread of the CTA; s: a word per warp.
__device__ __forceinline__ int64_t split_max_rows(const AttendArg& a, int heads, int group, int64_t* s) {
    int64_t ctas = 0;
    for (int r = threadIdx.x; r < a.R; r += blockDim.x) {
        const int64_t n = max(0, min(__ldg(a.cu + r + 1), a.T) - min(max(__ldg(a.cu + r), 0), a.T)), rows = n * group;
        if (rows >= PROMPT_MIN_ROWS) ctas += (rows + PROMPT_PAIR_ROWS - 1) / PROMPT_PAIR_ROWS * heads;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ctas += __shfl_xor_sync(0xffffffffu, ctas, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = ctas;
    __syncthreads();
    ctas = 0;
    for (int i = 0; i < (int)blockDim.x / 32; i++) ctas += s[i];
    __syncthreads();
    return ctas >= PROMPT_MIN_CTAS ? PROMPT_MIN_ROWS - 1 : INT64_MAX;
}
#endif

int split_tile_tokens(int dim);    // tokens of a tile
size_t split_part_bytes(int dim);  // workspace of one CTA
cudaError_t launch_split(const KvMaps& maps, const KvArg& kv, const AttendArg& a, const SplitWs& ws, int sms, int nr,
                         uint32_t type, int code, cudaStream_t s);

// The prompt kernel, for head_dim 64 and 128.
cudaError_t launch_prompt(const KvMaps& maps, const KvArg& kv, const AttendArg& a, uint32_t type, int code, cudaStream_t s);

}  // namespace rmoe
