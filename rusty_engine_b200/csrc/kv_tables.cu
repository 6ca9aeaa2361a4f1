// kv_tables.cu -- block tables and slot maps of the paged cache, built on the GPU from request
// lengths (rmoe_kv_extend), and giving blocks back (rmoe_kv_release).
//
// extend is three prefix sums over the requests (new tokens, new blocks, and which requests the
// free stack still covers) and then one independent step per token.  The sums are a few hundred
// additions, the tokens a few MB at most, so a launch boundary between the two would cost more
// than the sums: every CTA forms all sums in its own shared memory and then fills its share of
// the tokens, in one launch.  Measured (B200): 8 requests 2.8 us on the device (lengths, two prefix
// sums, tokens: latency), 512 requests with 164 thousand tokens 5.6 us (calls in a graph).
#include "kv_impl.h"

namespace rmoe {

static constexpr int EXT_THREADS = 1024;
static constexpr uint32_t EXT_MAX_R = 16384;

// Exclusive prefix sums of one 64-bit value per thread over the CTA; total in `sum`.  warp_tot: 32
// words, those past the CTA's warps 0.
__device__ __forceinline__ int64_t warp_scan(int64_t x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}
__device__ __forceinline__ int64_t cta_scan(int64_t v, int64_t* warp_tot, int64_t& sum) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t x = warp_scan(v);
    __syncthreads();  // warp_tot may still be read from the previous call
    if (lane == 31) warp_tot[w] = x;
    __syncthreads();
    const int64_t t = warp_tot[lane], all = warp_scan(t);  // every warp scans the warps' totals
    sum = __shfl_sync(0xffffffffu, all, 31);
    return __shfl_sync(0xffffffffu, all - t, w) + x - v;
}

__global__ void __launch_bounds__(EXT_THREADS) kv_extend_kernel(rmoe_kv_extend_args a) {
    extern __shared__ int32_t sm[];
    int32_t* s_cu = sm;                // [R + 1] first token of each request
    int32_t* s_first = sm + a.R + 1;   // [R] blocks that earlier requests take, -1: refused
    __shared__ int64_t warp_tot[32];
    __shared__ int s_used;
    const int tid = threadIdx.x, R = (int)a.R, bs = (int)a.block_size, sh = 31 - __clz(bs);
    const int nth = blockDim.x, per = (R + nth - 1) / nth, r0 = min(R, tid * per), r1 = min(R, r0 + per);
    if (tid < 32) warp_tot[tid] = 0;
    pdl_trigger();
    pdl_wait();
    const int height = max(0, min(__ldg(a.n_free), (int)a.free_cap));
    if (tid == 0) s_used = 0;
    int64_t mine = 0, total = 0;
    for (int r = r0; r < r1; r++) mine += max(0, __ldg(a.new_lens + r));
    int64_t at = cta_scan(mine, warp_tot, total);
    auto need = [&](int r, int64_t first, int n) -> int64_t {  // blocks r asks for, -1: does not fit its row or T
        const int64_t len = max(0, __ldg(a.lens + r));
        if (len + n > (int64_t)a.max_blocks * bs || first + n > (int64_t)a.T) return -1;
        return ((len + n + bs - 1) >> sh) - ((len + bs - 1) >> sh);
    };
    int64_t asked = 0, c = at;
    for (int r = r0; r < r1; r++) {
        const int n = max(0, __ldg(a.new_lens + r));
        asked += max((int64_t)0, need(r, c, n));
        c += n;
    }
    int64_t all = 0, up = cta_scan(asked, warp_tot, all);
    int used = 0;
    c = at;
    for (int r = r0; r < r1; r++) {
        const int n = max(0, __ldg(a.new_lens + r));
        const int64_t b = need(r, c, n);
        const bool ok = b == 0 || (b > 0 && up + b <= height);
        s_cu[r] = (int32_t)min(c, (int64_t)0x7fffffff);
        s_first[r] = ok ? (int32_t)up : -1;
        if (ok && b > 0) used = (int)(up + b);
        if (blockIdx.x == 0) {
            a.cu[r] = s_cu[r];
            a.lens_out[r] = ok ? max(0, __ldg(a.lens + r)) + n : __ldg(a.lens + r);
        }
        up += max((int64_t)0, b);
        c += n;
    }
    if (used) atomicMax(&s_used, used);
    if (tid == 0) s_cu[R] = (int32_t)min(total, (int64_t)0x7fffffff);
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        a.cu[R] = s_cu[R];
        *a.n_free_out = __ldg(a.n_free) < 0 ? 0 : height - s_used;
    }
    for (uint64_t t = blockIdx.x * (uint64_t)nth + tid; t < a.T; t += gridDim.x * (uint64_t)nth) {
        int slot = -1, pos = 0;
        if ((int64_t)t < s_cu[R]) {
            int lo = 0, hi = R - 1;  // the last request whose first token is at or before t (and that has tokens)
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if ((int64_t)s_cu[mid] <= (int64_t)t) lo = mid; else hi = mid - 1;
            }
            const int r = lo, len = max(0, __ldg(a.lens + r));
            pos = len + (int)((int64_t)t - s_cu[r]);
            if (s_first[r] >= 0) {
                const int have = (len + bs - 1) >> sh, page = pos >> sh;
                int32_t* entry = a.table + (size_t)r * a.max_blocks + page;
                int block;
                if (page < have) {
                    block = *entry;
                } else {
                    block = __ldg(a.free_list + (height - 1 - s_first[r] - (page - have)));
                    if (pos == max(page << sh, len)) *entry = block;  // the block's first new token
                }
                slot = block < 0 ? -1 : (block << sh) + (pos & (bs - 1));
            }
        }
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
}

// One CTA: prefix sums of the blocks to give back, then a warp per request moves them.  It runs once
// when requests end: 8 requests of 500 tokens 4.6 us, 64 of 8192 8.4, 512 of 4096 23.5 (B200, in a graph).
__global__ void __launch_bounds__(EXT_THREADS) kv_release_kernel(rmoe_kv_release_args a) {
    extern __shared__ int32_t s_at[];  // [R] stack position of the request's first block, -1: not done
    __shared__ int64_t warp_tot[32];
    const int tid = threadIdx.x, R = (int)a.R, bs = (int)a.block_size;
    const int per = (R + EXT_THREADS - 1) / EXT_THREADS, r0 = min(R, tid * per), r1 = min(R, r0 + per);
    const int height = max(0, min(__ldg(a.n_free), (int)a.free_cap));
    auto held = [&](int r) {
        return __ldg(a.done + r) ? (int)min(((int64_t)max(0, a.lens[r]) + bs - 1) / bs, (int64_t)a.max_blocks) : 0;
    };
    int64_t mine = 0, total = 0;
    for (int r = r0; r < r1; r++) mine += held(r);
    int64_t at = height + cta_scan(mine, warp_tot, total);
    for (int r = r0; r < r1; r++) {
        s_at[r] = __ldg(a.done + r) ? (int32_t)min(at, (int64_t)0x7fffffff) : -1;
        at += held(r);
    }
    __syncthreads();
    const int lane = tid & 31;
    for (int r = tid >> 5; r < R; r += EXT_THREADS / 32) {
        if (s_at[r] < 0) continue;
        const int n = held(r);
        int32_t* row = a.table + (size_t)r * a.max_blocks;
        for (int i = lane; i < (int)a.max_blocks; i += 32) {
            if (i < n && (int64_t)s_at[r] + i < (int64_t)a.free_cap) a.free_list[s_at[r] + i] = row[i];
            row[i] = -1;
        }
        __syncwarp();
        if (lane == 0) a.lens[r] = 0;
    }
    if (tid == 0) *a.n_free_out = (int32_t)min(height + total, (int64_t)a.free_cap);
}

}  // namespace rmoe

using namespace rmoe;

static rmoe_status check_tables(uint32_t R, uint32_t max_blocks, uint32_t bs, uint32_t cap) {
    if (!block_size_ok(bs)) return fail(RMOE_ERR_UNSUPPORTED, "block size %u (16, 32, 64 or 128)", bs);
    if (R > EXT_MAX_R) return fail(RMOE_ERR_UNSUPPORTED, "%u requests (at most %u)", R, EXT_MAX_R);
    if ((uint64_t)max_blocks * bs > 0x7fffffffull) return fail(RMOE_ERR_UNSUPPORTED, "%u blocks of %u in a row", max_blocks, bs);
    if (cap > 0x7fffffffu / bs) return fail(RMOE_ERR_UNSUPPORTED, "%u blocks of %u", cap, bs);
    return RMOE_OK;
}

extern "C" {

rmoe_status rmoe_kv_extend(const rmoe_kv_extend_args* a, void* stream) {
    if (!a) return fail(RMOE_ERR_INVALID, "null arguments");
    if (rmoe_status s = check_tables(a->R, a->max_blocks, a->block_size, a->free_cap)) return s;
    if (a->T > 0x7fffffffu) return fail(RMOE_ERR_UNSUPPORTED, "%u tokens", a->T);
    if (!a->n_free || !a->cu || !a->n_free_out || (a->R && (!a->table || !a->lens || !a->new_lens || !a->lens_out)) ||
        (a->T && (!a->positions || !a->slots)) || (a->free_cap && !a->free_list))
        return fail(RMOE_ERR_INVALID, "kv extend: null pointer");
    if (a->lens_out == a->lens || a->n_free_out == a->n_free)
        return fail(RMOE_ERR_INVALID, "kv extend: lens_out / n_free_out alias their inputs");
    const size_t smem = (2 * (size_t)a->R + 1) * 4;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(kv_extend_kernel, 132 << 10, done);
    if (e != cudaSuccess) return cuda_fail(e, "kv extend");
    // small batches: fewer threads, whose barriers are shorter
    const unsigned nth = a->R <= 256 && a->T <= 16384 ? 256 : EXT_THREADS, grid = (unsigned)((a->T + nth - 1) / nth);
    e = launch_pdl(kv_extend_kernel, dim3(grid < 1 ? 1 : grid < 148 ? grid : 148), dim3(nth), smem,
                   static_cast<cudaStream_t>(stream), *a);
    return e == cudaSuccess ? RMOE_OK : cuda_fail(e, "kv extend launch");
}

rmoe_status rmoe_kv_release(const rmoe_kv_release_args* a, void* stream) {
    if (!a) return fail(RMOE_ERR_INVALID, "null arguments");
    if (rmoe_status s = check_tables(a->R, a->max_blocks, a->block_size, a->free_cap)) return s;
    if (!a->n_free || !a->n_free_out || (a->R && (!a->table || !a->lens || !a->done)) || (a->free_cap && !a->free_list))
        return fail(RMOE_ERR_INVALID, "kv release: null pointer");
    if (a->n_free_out == a->n_free) return fail(RMOE_ERR_INVALID, "kv release: n_free_out aliases n_free");
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(kv_release_kernel, 132 << 10, done);
    if (e != cudaSuccess) return cuda_fail(e, "kv release");
    kv_release_kernel<<<1, EXT_THREADS, (size_t)a->R * 4 + 4, static_cast<cudaStream_t>(stream)>>>(*a);
    e = cudaGetLastError();
    return e == cudaSuccess ? RMOE_OK : cuda_fail(e, "kv release launch");
}

}  // extern "C"
