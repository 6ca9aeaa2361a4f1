// kv_impl.h -- the paged 8-bit KV cache and rotary-position handles, shared by the translation
// units that implement their entry points (kv.cu, rope.cu, kv_append.cu, kv_attend.cu).
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

#include "layer_impl.h"

struct rmoe_rope {
    int device = 0;
    uint32_t rot = 0, layout = 0, max_pos = 0;
    float2* table = nullptr;  // [max_pos][rot / 2] (cos, sin), owned
    unsigned* status = nullptr;
    rmoe::Owned own;
};

namespace rmoe {
struct KvMaps {
    CUtensorMap k, v;  // the codes as rows of head_dim bytes (make_code_map)
};

// Workspace of the split kernel: two (M, l, O) pieces per CTA, and a count per CTA that is 0
// between calls.
struct SplitWs {
    float* part;
    unsigned* ticket;
};

// The workspaces of a cache.  Calls on one stream follow one another and share one; calls on
// different streams may run at the same time and have one each.  So have the calls that a stream
// captures: their graph may run beside the stream's own later calls.
struct SplitSlot {
    enum Use { FREE, CALLS, GRAPHS } use;
    unsigned long long stream;  // CALLS: its id, which no later stream of the process gets; GRAPHS: its handle
    SplitWs ws;                 // one allocation, at part
};
static constexpr int MAX_SPLIT_SLOTS = 64;
}  // namespace rmoe

struct rmoe_kv {
    int device = 0;
    uint32_t n_blocks = 0, bs = 0, heads = 0, dim = 0, code = 0;
    uint8_t *k = nullptr, *v = nullptr;
    float *ks = nullptr, *vs = nullptr;
    unsigned* status = nullptr;
    rmoe::KvMaps split_maps{};     // boxes of a split-kernel tile
    rmoe::KvMaps prompt_maps{};    // boxes of a prompt-kernel tile: a block
    int sms = 0;
    std::mutex slots_mu;
    rmoe::SplitSlot slots[rmoe::MAX_SPLIT_SLOTS]{};
    int n_slots = 0;
    rmoe::Owned own;

    rmoe_kv() = default;
    ~rmoe_kv() {
        for (int i = 0; i < n_slots; i++) cudaFree(slots[i].ws.part);
    }
};

namespace rmoe {

// Heads of T tokens as the kernels take them (rmoe_rows without the padding).
struct Rows {
    char* p;
    int64_t st, sh;  // strides of a token and of a head, in elements
    int heads;
    bool vec;        // data and strides are multiples of 16 bytes
};

// Whether `device` exists (a handle made on it would otherwise land on the current device).
inline rmoe_status check_device(int32_t device) {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess) {
        cudaGetLastError();  // not sticky: the next launch check must not see it
        return fail(RMOE_ERR_CUDA, "no CUDA device");
    }
    return device >= 0 && device < n ? RMOE_OK : fail(RMOE_ERR_INVALID, "device %d out of range", device);
}

// Raises a kernel's dynamic shared-memory limit on the current device, the first time only (a call
// of its own took longer than the launch).
template <typename K>
inline cudaError_t allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_relaxed) & bit))) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// Has a kernel's launches ask for the largest shared memory of an SM, whatever they use of it.
template <typename K>
inline cudaError_t all_shared(K kernel, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_relaxed) & bit))) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

inline uint32_t elt_size(uint32_t type) { return type == T_F32 ? 4 : 2; }
inline bool elt_ok(uint32_t type) { return type == T_F32 || type == T_F16 || type == T_BF16; }

// Checks one rmoe_rows argument and fills r; `what` names it in the message.
rmoe_status check_rows(const rmoe_rows& a, uint32_t T, uint32_t type, const char* what, Rows& r);

// What the kernels need of a rope handle.
struct RopeArg {
    const float2* table;  // null: no rotation
    const int32_t* pos;
    int rot, half, max_pos;
    float sign;           // -1 turns back
};

// The cache as the kernels take it.
struct KvArg {
    uint8_t *k, *v;
    float *ks, *vs;
    int n_blocks, bs, heads, dim;  // bs a power of two
    unsigned* status;
    int shift;                     // log2 bs
};
inline KvArg kv_arg(const rmoe_kv* kv) {
    return KvArg{kv->k, kv->v, kv->ks, kv->vs, (int)kv->n_blocks, (int)kv->bs, (int)kv->heads, (int)kv->dim, kv->status,
                 kv->bs == 16 ? 4 : kv->bs == 32 ? 5 : kv->bs == 64 ? 6 : 7};
}
inline bool block_size_ok(uint32_t bs) { return bs == 16 || bs == 32 || bs == 64 || bs == 128; }

cudaError_t launch_rope_apply(const Rows& q, const Rows& qo, const Rows& k, const Rows& ko, const RopeArg& ra, int T,
                              int dim, uint32_t type, unsigned* status, cudaStream_t s);

}  // namespace rmoe
