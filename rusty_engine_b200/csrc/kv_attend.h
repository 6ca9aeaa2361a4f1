// kv_attend.h -- the attention kernels' arguments and launchers (kv_attend.cu chooses).
#pragma once
#include "kv_impl.h"

namespace rmoe {

struct AttendArg {
    Rows q, out;
    const int32_t *table, *lens, *cu;
    float* lse;
    int R, max_blocks, T;
    float scale;
    int window;
    int64_t split_rows;  // requests of more rows (new tokens x query heads per kv head) are another kernel's
};

// Workspace of the split kernel: two (M, l, O) pieces per CTA, and a count per CTA that is 0
// between calls.
struct SplitWs {
    float* part;
    unsigned* ticket;
};

int split_tile_tokens(int dim);    // tokens of a tile
size_t split_part_bytes(int dim);  // workspace of one CTA
cudaError_t launch_split(const KvMaps& maps, const KvArg& kv, const AttendArg& a, const SplitWs& ws, int sms, int nr,
                         uint32_t type, int code, cudaStream_t s);

}  // namespace rmoe
