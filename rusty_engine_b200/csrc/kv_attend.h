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

// Workspace of the split kernel: two (M, l, O) pieces per CTA, and a count per CTA that is 0
// between calls.
struct SplitWs {
    float* part;
    unsigned* ticket;
};

// Rows of a request: its new tokens x the query heads that share a kv head.
static constexpr int PROMPT_MIN_ROWS = 64, PROMPT_PAIR_ROWS = 256, PROMPT_MIN_CTAS = 24;

#ifdef __CUDACC__
// The most rows of a request that the split kernel takes when the prompt kernel runs too.  The
// prompt kernel works on 256 rows per CTA at ten times the split kernel's rate, but does not split
// the keys: with fewer CTAs than a tenth of the chip the split kernel, which always fills it, is
// the faster one.  Called by every thread of the CTA; s: a word per warp.
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
