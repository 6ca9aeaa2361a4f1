// kv_prompt.cu -- attention over the 8-bit paged cache for many query rows: prompts and chunks of
// them, on the tensor cores (tcgen05).  head_dim 64 and 128.
//
// Mathematics: as in kv_split.cu,  out = sum_j 2^(x_j - M) vc_j / sum_j 2^(x_j - M) / vs_j  with
// x_j = scale log2(e) ks_j q.kc_j + log2(vs_j).  A row may be any (token, query head) of the kv
// head, so the rows of a CTA are 128-row tiles of consecutive (token, head of the group).
//
// Roles of the CTA's 16 warps: one brings raw 8-bit tiles of 128 keys by TMA, four widen them to
// fp16 operand tiles (128-byte swizzle; K as the K-major and V as the MN-major operand, both in
// the cache's own [key][element] order), one issues the products, and eight read S out of tensor
// memory, one row per thread.
//   16-bit calls: two row tiles share every K / V tile (the widening is paid once for 256 rows);
//     while one tile's softmax runs, the other's products do.  P goes back to tensor memory as
//     fp16 over its own S and is the A operand from there.  O stays in tensor memory; it is only
//     rescaled when a row's maximum grew by more than 2^LAG, by the softmax threads.
//     P is carried as 2^UP times itself, so a weight has its 11 bits down to 2^-21 of the row's largest
//     (2^-29 when M lags behind that).
//   f32 calls: q and P (2^15 times itself) are fp16 pairs (hi + lo, twice the products), one row tile, S in
//     two buffers (head_dim 128: 92 bytes a thread spill).  The tensor cores cut every partial sum short, about 2^-24 per step and all one
//     way, which over a long row is more than f32 attention may lose (up to 4.5e-6 measured); so each key
//     tile has its own O in tensor memory, and the other four warps add the tiles up in registers.
//
// Measured (B200): 4096 new and 3 decoded tokens over up to 8192 keys, 32 heads over 4 kv heads of
// 128, bf16, int8 cache: 480 to 493 us on changing inputs (462 when one input repeats), 412.6 GFLOP, 837 to 860
// TFLOP/s = 51 to 52% of the cuBLAS rate; a 2048-token prompt in f32: 122 us (120), 34.4 GFLOP, 281 TFLOP/s (twice
// that with the pairs' products), in bf16 63 us, 545 TFLOP/s; 64 wide 92 and 48 us.  No pipe is full (tensor
// and special functions 47% each in the mixed batch in bf16): softmax, P V and the next S of a row tile follow one another, and
// only the other row tile's work hides them.  More row tiles do not fit: S and O of two fill tensor
// memory's 512 columns at head_dim 128.
#include "kv_attend.h"
#include "kv_widen.cuh"
#include "rope.cuh"
#include "tc_ptx.cuh"

namespace rmoe {

static constexpr int PT = 512;    // threads
static constexpr int PKV = 128;   // keys per tile

template <int D, bool PAIR>
struct PromptShape {
    static constexpr int NRT = PAIR ? 1 : 2;             // row tiles
    // M may lag behind a row's maximum by LAG, and the weights are carried as 2^UP times themselves:
    // together they reach 2^15 at most.  A shorter lag keeps more of small weights but rescales O more
    // often (4096 new tokens in bf16: 8 466.6 us, 5 482.6, 3 493.7)
    static constexpr int LAG = PAIR ? 0 : 8, UP = 15 - LAG;
    static constexpr float DOWN = 1.0f / (1 << UP);
    static constexpr int QB = 128 * D * 2;               // fp16 bytes of a Q, K or V tile
    static constexpr int RAW = PKV * D;
    // operand buffers; f32 has room for three: K's is free again as soon as S is made, V's only after P V
    static constexpr int KN = PAIR ? 1 : 2, VN = 2;
    static constexpr int Q0 = 0, K0 = 2 * QB, V0 = K0 + KN * QB, R0 = V0 + VN * QB, END = R0 + 2 * RAW;
    static constexpr int SMEM = END + 1024;              // + alignment
};

struct PromptBars {
    uint64_t q_full, raw_full[2], raw_empty[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_half[2], p_full[2], o_full[2],
        o_empty[2], meta_full[4], drain;
};

// Registers a thread of this warpgroup (all four warps execute it).
template <int N> __device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N> __device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }

// Two f32 in one register pair.
__device__ __forceinline__ uint64_t f2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void un2(uint64_t r, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(x), "=f"(y) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// The factor from a product of codes to the exponent: positive, so that -infinity stays it.
__device__ __forceinline__ float score_scale(float qs, float ks) { return fmaxf(qs * ks, 1.17549435e-38f); }

template <typename T, int CODE, int D>
__global__ void __launch_bounds__(PT, 1)
kv_prompt_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, KvArg kv, AttendArg a) {
    constexpr bool PAIR = sizeof(T) == 4;
    using S = PromptShape<D, PAIR>;
    constexpr int NRT = S::NRT, KN = S::KN, VN = S::VN, CH = D / 32;
    extern __shared__ uint8_t smem_raw[];
    __shared__ PromptBars bars;
    __shared__ uint32_t s_tmem;
    __shared__ int64_t s_sum[PT / 32];
    __shared__ int s_req[2];
    __shared__ float4 s_meta[4][PKV / 16];                // per 16 keys: K scale, log2 V scale, 1 / V scale, 1: no such block
    __shared__ float s_alpha[PAIR ? 4 : 1][PAIR ? 128 : 1];  // f32: what the earlier tiles' O is multiplied by
    __shared__ float s_fin[2][PAIR ? 128 : 1];            // f32: M and l of the rows

    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, wg = w >> 2;
    const int heads = kv.heads, bs = kv.bs, group = a.group;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;

    pdl_wait();
    pdl_trigger();  // the split kernel, which takes the other requests, fills the SMs that run out of work here
    // ---- which request, head and rows ----
    const int64_t max_rows = split_max_rows(a, heads, group, s_sum);
    if (max_rows == INT64_MAX) return;
    auto rows_of = [&](int r) -> int64_t {
        const int q0 = min(max(__ldg(a.cu + r), 0), a.T);
        return (int64_t)max(0, min(__ldg(a.cu + r + 1), a.T) - q0) * group;
    };
    auto items_of = [&](int r) -> int64_t {
        const int64_t rows = rows_of(r);
        return rows > max_rows ? (rows + NRT * 128 - 1) / (NRT * 128) * heads : 0;
    };
    {
        const int per = (a.R + PT - 1) / PT, r0 = min(a.R, tid * per), r1 = min(a.R, r0 + per);
        int64_t mine = 0;
        for (int r = r0; r < r1; r++) mine += items_of(r);
        int64_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) s_sum[w] = incl;
        if (tid == 0) s_req[0] = -1;
        __syncthreads();
        int64_t before = 0;
        for (int i = 0; i < w; i++) before += s_sum[i];
        int64_t at = before + incl - mine, me = blockIdx.x;
        if (me >= at && me < at + mine) {
            int r = r0;
            while (me >= at + items_of(r)) at += items_of(r++);
            s_req[0] = r;
            s_req[1] = (int)(items_of(r) - 1 - (me - at));  // the request's last rows, which see most, first
        }
        __syncthreads();
    }
    const int r = s_req[0];
    if (r < 0) return;
    const int kh = s_req[1] % heads, row0 = s_req[1] / heads * (NRT * 128);
    const int q0 = min(max(__ldg(a.cu + r), 0), a.T), n = max(0, min(__ldg(a.cu + r + 1), a.T) - q0);
    const int len = __ldg(a.lens + r), pos0 = len - (__ldg(a.cu + r + 1) - __ldg(a.cu + r));
    const int hi = (int)min((int64_t)max(len, 0), (int64_t)a.max_blocks * bs);
    const int tok_last = min(n - 1, (row0 + NRT * 128 - 1) / group);
    const int kmax = min(pos0 + tok_last + 1, hi), kmin = first_seen(a.window, pos0 + row0 / group);
    const int jt0 = kmin / PKV, nt = kmax > kmin ? (kmax + PKV - 1) / PKV - jt0 : 0;  // key tiles

    if (tid == 0) {
        tc::mbar_init(smem_u32(&bars.q_full), 4 * NRT);
        for (int i = 0; i < 2; i++) {
            tc::mbar_init(smem_u32(&bars.raw_full[i]), 1);
            tc::mbar_init(smem_u32(&bars.raw_empty[i]), 4);
            tc::mbar_init(smem_u32(&bars.k_full[i]), 4);
            tc::mbar_init(smem_u32(&bars.k_empty[i]), 1);
            tc::mbar_init(smem_u32(&bars.v_full[i]), 4);
            tc::mbar_init(smem_u32(&bars.v_empty[i]), 1);
            tc::mbar_init(smem_u32(&bars.s_full[i]), 1);
            tc::mbar_init(smem_u32(&bars.p_half[i]), 4);
            tc::mbar_init(smem_u32(&bars.p_full[i]), 4);
            tc::mbar_init(smem_u32(&bars.o_full[i]), 1);
            tc::mbar_init(smem_u32(&bars.o_empty[i]), 4);
        }
        for (int i = 0; i < 4; i++) tc::mbar_init(smem_u32(&bars.meta_full[i]), 1);
        tc::mbar_init(smem_u32(&bars.drain), 1);
        tc::fence_mbar_init();
    }
    if (w == 13) tc::tmem_alloc(smem_u32(&s_tmem), 512);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tm = s_tmem;
    // tensor memory columns: S (and P) of tile / buffer i at 128 i, O at 256 + 128 i
    bool dead = false;
    auto wait = [&](uint64_t& b, uint32_t parity) {  // by whole warps: all lanes go on, or none
        if (!dead) dead = !__all_sync(0xffffffffu, tc::mbar_wait_tries(smem_u32(&b), parity & 1));
        return !dead;
    };

    // Registers go to the roles that hold rows: 192 + 192 + 72 + 56 a thread (f32: 184 + 184 + 80 +
    // 64), of 128 x 4 at launch.  Each role's branch begins with its warpgroup's share.
    if (wg == 3) {
        reg_dec<PAIR ? 64 : 56>();
        if (w == 12) {
            // ---- producer: raw tiles and the scales of their blocks ----
            const int br = min(bs, PKV), nb = PKV / br;
            auto lookup = [&](int j) {
                const int t = (jt0 + j) * PKV + 16 * lane;
                return j < nt && lane < 8 && t < kmax ? __ldg(a.table + (int64_t)r * a.max_blocks + (t >> kv.shift)) : -1;
            };
            int blk = lookup(0), issued = 0;
            for (int j = 0; j < nt; j++) {
                const int t = (jt0 + j) * PKV + 16 * lane;
                const bool want = lane < 8 && t < kmax, ok = want && (unsigned)blk < (unsigned)kv.n_blocks;
                // (a block whose keys all lie before the window may have been given back)
                if (want && !ok && t + 16 > kmin) atomicOr(kv.status, (unsigned)DERR_INDEX);
                const int64_t bh = ok ? (int64_t)blk * heads + kh : 0;
                const float ks = ok ? __ldg(kv.ks + bh) : 0.0f, vs = ok ? __ldg(kv.vs + bh) : 1.0f;
                const int next = lookup(j + 1);
                // lane b < nb: the box of block rows at key b * br
                const int src = lane < nb ? lane * br / 16 : 0;
                const int bblk = __shfl_sync(0xffffffffu, blk, src);
                const bool bok = __shfl_sync(0xffffffffu, (int)ok, src) && lane < nb;
                const unsigned mask = __ballot_sync(0xffffffffu, bok);
                const int row = bok ? (int)(((int64_t)bblk * heads + kh) * bs) : 0;
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    if (j > 0 && !wait(bars.raw_empty[v], j - 1)) break;
                    const uint32_t bar = smem_u32(&bars.raw_full[v]);
                    if (lane == 0) tc::mbar_arrive_expect_tx(bar, __popc(mask) * br * D);
                    __syncwarp();
                    if (bok) tc::tma_2d(base + S::R0 + v * S::RAW + lane * br * D, v ? &vmap : &kmap, 0, row, bar);
                    issued++;
                }
                if (dead) break;
                if (lane < 8) {
                    const float f = v_scale_floor(vs);
                    s_meta[j & 3][lane] = make_float4(ks, log2f(f), 1.0f / f, ok ? 0.0f : 1.0f);
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(smem_u32(&bars.meta_full[j & 3]));
                blk = next;
            }
            if (dead)  // let the copies in flight land
                for (int v = 0; v < 2; v++) {
                    const int c = (issued + 1 - v) / 2;  // copies into buffer v
                    if (c > 0) tc::mbar_wait(smem_u32(&bars.raw_full[v]), (c - 1) & 1);
                }
        } else if (w == 13) {
            // ---- products ----
            if (nt > 0) {
                const uint32_t lead = lane == 0;
                constexpr uint32_t idS = tc::idesc_f16(128, PKV), idO = tc::idesc_f16(128, D) | tc::IDESC_B_MN;
                const uint64_t qd = tc::smem_desc_sw128(base + S::Q0), kd = tc::smem_desc_sw128(base + S::K0),
                               vd = tc::smem_desc_mn_sw128(base + S::V0, PKV * 128);
                const uint32_t dh = (uint32_t)(kd >> 32), vh = (uint32_t)(vd >> 32);
                auto mma_s = [&](int q, uint32_t d, int buf) {  // S = Q K^T; q: the Q tile (lo half next to it)
                    const uint32_t qa = (uint32_t)qd + q * (S::QB >> 4), kb = (uint32_t)kd + buf * (S::QB >> 4);
#pragma unroll
                    for (int half = PAIR ? 1 : 0; half >= 0; half--)
#pragma unroll
                        for (int k = 0; k < D / 16; k++) {
                            const uint32_t off = ((k / 4) * 16384 + (k % 4) * 32) >> 4;
                            tc::mma_ss_lead(lead, d, qa + (half * (S::QB >> 4) + off), dh, kb + off, dh, idS, k > 0 || (PAIR && half == 0));
                        }
                };
                auto mma_o = [&](uint32_t d, uint32_t p, int buf, uint32_t add, int part) {  // O (+)= P V of half the keys
                    const uint32_t vb = (uint32_t)vd + buf * (S::QB >> 4) + part * (4 * 2048 >> 4);
                    p += part * 64;
#pragma unroll
                    for (int half = PAIR ? 1 : 0; half >= 0; half--)
#pragma unroll
                        for (int k = 0; k < PKV / 32; k++)
                            tc::mma_ts_lead(lead, d, p + (k / 2) * 32 + (k % 2) * 8 + half * 16, vb + (k * 2048 >> 4), vh, idO,
                                            k > 0 || (PAIR && half == 0) ? 1u : add);
                };
                if (wait(bars.q_full, 0) && wait(bars.k_full[0], 0)) {
                    tc::fence_after_sync();
                    for (int t = 0; t < NRT; t++) {
                        mma_s(t, tm + t * 128, 0);
                        tc::mma_commit_lead(lead, smem_u32(&bars.s_full[t]));
                    }
                    tc::mma_commit_lead(lead, smem_u32(&bars.k_empty[0]));
                }
                for (int j = 0; j < nt && !dead; j++) {
                    if (PAIR) {
                        if (j + 1 < nt) {
                            if (!wait(bars.k_full[(j + 1) % KN], (j + 1) / KN)) break;
                            tc::fence_after_sync();
                            mma_s(0, tm + ((j + 1) & 1) * 128, (j + 1) % KN);
                            tc::mma_commit_lead(lead, smem_u32(&bars.s_full[(j + 1) & 1]));
                            tc::mma_commit_lead(lead, smem_u32(&bars.k_empty[(j + 1) % KN]));
                        }
                        if (!wait(bars.v_full[j % VN], j / VN) || !wait(bars.p_half[j & 1], j / 2)) break;
                        if (j >= 2 && !wait(bars.o_empty[j & 1], j / 2 - 1)) break;
                        tc::fence_after_sync();
                        mma_o(tm + 256 + (j & 1) * 128, tm + (j & 1) * 128, j % VN, 0, 0);
                        if (!wait(bars.p_full[j & 1], j / 2)) break;
                        tc::fence_after_sync();
                        mma_o(tm + 256 + (j & 1) * 128, tm + (j & 1) * 128, j % VN, 1, 1);
                        tc::mma_commit_lead(lead, smem_u32(&bars.o_full[j & 1]));
                        tc::mma_commit_lead(lead, smem_u32(&bars.v_empty[j % VN]));
                    } else {
                        for (int t = 0; t < NRT; t++) {
                            if (t == 0 && !wait(bars.v_full[j % VN], j / VN)) break;
                            if (!wait(bars.p_half[t], j)) break;
                            tc::fence_after_sync();
                            mma_o(tm + 256 + t * 128, tm + t * 128, j % VN, j > 0, 0);
                            if (!wait(bars.p_full[t], j)) break;
                            tc::fence_after_sync();
                            mma_o(tm + 256 + t * 128, tm + t * 128, j % VN, 1, 1);
                            tc::mma_commit_lead(lead, smem_u32(&bars.o_full[t]));
                            if (t == NRT - 1) tc::mma_commit_lead(lead, smem_u32(&bars.v_empty[j % VN]));
                            if (j + 1 < nt) {
                                if (t == 0 && !wait(bars.k_full[(j + 1) % KN], (j + 1) / KN)) break;
                                tc::fence_after_sync();
                                mma_s(t, tm + t * 128, (j + 1) % KN);
                                tc::mma_commit_lead(lead, smem_u32(&bars.s_full[t]));
                                if (t == NRT - 1) tc::mma_commit_lead(lead, smem_u32(&bars.k_empty[(j + 1) % KN]));
                            }
                        }
                    }
                }
                tc::mma_commit_lead(lead, smem_u32(&bars.drain));  // nothing may run into freed tensor memory
                if (!__all_sync(0xffffffffu, tc::mbar_wait(smem_u32(&bars.drain), 0))) dead = true;
            }
        }
    } else if (wg == 2) {
        // ---- widening: one key per thread ----
        reg_dec<PAIR ? 80 : 72>();
        const int row = tid - 256;
        for (int j = 0; j < nt; j++) {
            if (!wait(bars.meta_full[j & 3], j >> 2)) break;
            const int key = (jt0 + j) * PKV + row;
            // keys that no row sees may hold anything, NaN codes too, and 0 * NaN is NaN
            const bool live = key < kmax && key >= kmin && s_meta[j & 3][row >> 4].w == 0.0f;
#pragma unroll 1
            for (int v = 0; v < 2; v++) {
                const int nbuf = v ? VN : KN, b = j % nbuf;
                if (!wait(bars.raw_full[v], j)) break;
                if (j >= nbuf && !wait(v ? bars.v_empty[b] : bars.k_empty[b], j / nbuf - 1)) break;
                const uint32_t src = base + S::R0 + v * S::RAW, dst = base + (v ? S::V0 : S::K0) + b * S::QB + row * 128;
                uint4 x[D / 16];
#pragma unroll
                for (int c = 0; c < D / 16; c++)
                    x[c] = D == 64 ? lds128(src + row * 64 + ((c ^ ((row >> 1) & 3)) << 4)) : lds128(src + row * 128 + ((c ^ (row & 7)) << 4));
                if (!__all_sync(0xffffffffu, live) && !live)
#pragma unroll
                    for (int c = 0; c < D / 16; c++) x[c] = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int c = 0; c < D / 16; c++) {
                    uint32_t y[8];
                    widen4<CODE>(x[c].x, y[0], y[1]);
                    widen4<CODE>(x[c].y, y[2], y[3]);
                    widen4<CODE>(x[c].z, y[4], y[5]);
                    widen4<CODE>(x[c].w, y[6], y[7]);
                    const uint32_t d = dst + (c / 4) * 16384;
                    sts128(d + (((2 * c & 7) ^ (row & 7)) << 4), make_uint4(y[0], y[1], y[2], y[3]));
                    sts128(d + (((2 * c + 1 & 7) ^ (row & 7)) << 4), make_uint4(y[4], y[5], y[6], y[7]));
                }
                tc::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tc::mbar_arrive(smem_u32(v ? &bars.v_full[b] : &bars.k_full[b]));
                    tc::mbar_arrive(smem_u32(&bars.raw_empty[v]));
                }
            }
            if (dead) break;
        }
    } else {
        reg_inc<PAIR ? 184 : 192>();
        const int rt = PAIR ? 0 : wg, lrow = tid & 127;
        const uint32_t tl = tm + ((uint32_t)((w & 3) * 32) << 16);
        const int row = row0 + rt * 128 + lrow, tok = row / group, h = kh * group + row % group;
        const bool live = tok < n;
        T* op = reinterpret_cast<T*>(a.out.p) + (int64_t)(q0 + (live ? tok : 0)) * a.out.st + (int64_t)h * a.out.sh;
        auto finish = [&](int c, const float* v, float l) {  // 32 elements of the row
            const float inv = l > 0.0f ? S::DOWN / l : (l == 0.0f ? 0.0f : l);
            float y[32];
#pragma unroll
            for (int i = 0; i < 32; i++) y[i] = l == 0.0f ? 0.0f : v[i] * inv;
            if (live)
#pragma unroll
                for (int i = 0; i < 4; i++) store8(op + c * 32 + i * 8, a.out.vec, y + i * 8);
        };
        auto put_lse = [&](float m, float l) {
            if (live && a.lse) a.lse[(int64_t)(q0 + tok) * a.q.heads + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
        };
        if (PAIR && wg == 1) {
            // ---- f32: adding up the tiles' O ----
            float acc[D];
#pragma unroll
            for (int i = 0; i < D; i++) acc[i] = 0.0f;
            for (int j = 0; j < nt; j++) {
                if (!wait(bars.o_full[j & 1], j / 2)) break;
                tc::fence_after_sync();
                const float al = s_alpha[PAIR ? j & 3 : 0][PAIR ? lrow : 0];
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    uint32_t v[32];
                    tc::tmem_ld32(tl + 256 + (j & 1) * 128 + c * 32, v);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; i++) acc[c * 32 + i] = fmaf(acc[c * 32 + i], al, __uint_as_float(v[i]));
                }
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(smem_u32(&bars.o_empty[j & 1]));
            }
            if (!dead) {
                const float l = nt > 0 ? s_fin[1][PAIR ? lrow : 0] : 0.0f;
#pragma unroll
                for (int c = 0; c < CH; c++) finish(c, acc + c * 32, l);
                put_lse(nt > 0 ? s_fin[0][PAIR ? lrow : 0] : 0.0f, l);
            }
        } else {
            // ---- q to operand tiles ----
            const T* qp = reinterpret_cast<const T*>(a.q.p) + (int64_t)(q0 + (live ? tok : 0)) * a.q.st + (int64_t)h * a.q.sh;
            // the whole row at once: loads one after the other took 12 thousand cycles
            float v0[D], mx = 0.0f;
            if (a.q.vec) {
                constexpr int W = 16 / sizeof(T);
#pragma unroll
                for (int c = 0; c < D / W; c++) {
                    T y[W];
                    *reinterpret_cast<uint4*>(y) = *(reinterpret_cast<const uint4*>(qp) + c);
#pragma unroll
                    for (int i = 0; i < W; i++) v0[c * W + i] = Elt<T>::get(y[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < D; i++) v0[i] = Elt<T>::get(qp[i]);
            }
#pragma unroll
            for (int i = 0; i < D; i++) {
                if (!live) v0[i] = 0.0f;
                mx = fmaxf(mx, fabsf(v0[i]));
            }
            const int e = q_exponent(mx);
            // the sign of the scale goes to q, and a scale of 0 makes q 0: qs is positive
            const float dn = exp2i(-e) * (a.scale < 0.0f ? -1.0f : a.scale == 0.0f ? 0.0f : 1.0f);
            const float qs = exp2i(e) * (a.scale == 0.0f ? 1.0f : fabsf(a.scale)) * LOG2E;
#pragma unroll
            for (int c = 0; c < D / 8; c++) {
                uint32_t hh[4], ll[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x = v0[c * 8 + 2 * i] * dn, y = v0[c * 8 + 2 * i + 1] * dn;
                    hh[i] = pack_f16x2(x, y);
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hh[i]));
                    ll[i] = pack_f16x2(x - f.x, y - f.y);
                }
                const uint32_t d = base + S::Q0 + rt * S::QB + (c / 8) * 16384 + lrow * 128 + (((c & 7) ^ (lrow & 7)) << 4);
                sts128(d, make_uint4(hh[0], hh[1], hh[2], hh[3]));
                if (PAIR) sts128(d + S::QB, make_uint4(ll[0], ll[1], ll[2], ll[3]));
            }
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(smem_u32(&bars.q_full));
            // ---- softmax ----
            const int vhi = live ? min(pos0 + tok + 1, hi) : 0, vlo = first_seen(a.window, pos0 + tok);
            // keys that every row of the tile sees
            const int first = (row0 + rt * 128) / group, last = min(n - 1, (row0 + rt * 128 + 127) / group);
            const int all_hi = min(pos0 + first + 1, hi), all_lo = first_seen(a.window, pos0 + last);
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; j < nt; j++) {
                const int sb = PAIR ? j & 1 : rt, key0 = (jt0 + j) * PKV;
                const uint32_t sp = tl + sb * 128;
                if (!wait(bars.meta_full[j & 3], j >> 2)) break;
                const float4* meta = s_meta[j & 3];
                bool masked = key0 < all_lo || key0 + PKV > all_hi;
#pragma unroll
                for (int i = 0; i < 8; i++) masked |= meta[i].w != 0.0f;
                if (!wait(bars.s_full[sb], PAIR ? j / 2 : j)) break;
                tc::fence_after_sync();
                // the row of S, masked where a key is not this row's
                uint32_t v[PKV];
#pragma unroll
                for (int c = 0; c < 4; c++) tc::tmem_ld32(sp + c * 32, v + c * 32);
                tc::tmem_ld_wait();
                if (masked) {
#pragma unroll
                    for (int g = 0; g < 8; g++) {
                        const bool gone = meta[g].w != 0.0f;
                        const int b = gone ? 0 : vhi - (key0 + 16 * g), t = vlo - (key0 + 16 * g);  // keys t .. b - 1 of the 16
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (i >= b || i < t) v[g * 16 + i] = 0xff800000u;  // -infinity
                        asm volatile("" ::: "memory");  // a branch: few tiles are masked
                    }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int g = 0; g < 8; g++) {
                    const float4 mt = meta[g];
                    float x[2] = {__uint_as_float(v[g * 16]), __uint_as_float(v[g * 16 + 1])};
#pragma unroll
                    for (int i = 2; i < 16; i++) x[i & 1] = fmaxf(x[i & 1], __uint_as_float(v[g * 16 + i]));
                    mx = fmaxf(mx, fmaf(fmaxf(x[0], x[1]), score_scale(qs, mt.x), mt.y));
                }
                const bool grow = mx > m + (float)S::LAG;
                const float mn = grow ? mx : m, mu = mn == -INFINITY ? 0.0f : mn;
                const float al = grow ? ex2(m - mu) : 1.0f;
                if (PAIR) {
                    s_alpha[PAIR ? j & 3 : 0][PAIR ? lrow : 0] = al;
                } else if (j > 0 && __any_sync(0xffffffffu, grow && m != -INFINITY)) {
                    if (!wait(bars.o_full[rt], j - 1)) break;
                    tc::fence_after_sync();
#pragma unroll
                    for (int c = 0; c < CH * 2; c++) {
                        uint32_t o[16];
                        tc::tmem_ld16(tl + 256 + rt * 128 + c * 16, o);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * al);
                        tc::tmem_st16(tl + 256 + rt * 128 + c * 16, o);
                    }
                }
                m = mn;
                l *= al;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t ph[16], pl[16];
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        const float4 mt = meta[2 * c + g];
                        const float sc = score_scale(qs, mt.x), off = mt.y - mu + (float)S::UP;
                        const uint64_t sc2 = f2(sc, sc), off2 = f2(off, off);
                        uint64_t sum = 0;
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const int e = c * 32 + g * 16 + 2 * i;
                            float x, y;
                            un2(fma2(f2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), sc2, off2), x, y);
                            x = ex2(x);
                            y = ex2(y);
                            sum = add2(sum, f2(x, y));
                            const uint32_t hh = pack_f16x2(x, y);
                            ph[g * 8 + i] = hh;
                            if (PAIR) {
                                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hh));
                                pl[g * 8 + i] = pack_f16x2(x - f.x, y - f.y);
                            }
                        }
                        float x, y;
                        un2(sum, x, y);
                        l = fmaf((x + y) * S::DOWN, mt.z, l);
                    }
                    tc::tmem_st16(sp + c * 32, ph);
                    if (PAIR) tc::tmem_st16(sp + c * 32 + 16, pl);
                    if (c == 1) {  // the products of the first half of the keys can begin
                        tc::tmem_st_wait();
                        tc::fence_before_sync();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(smem_u32(&bars.p_half[sb]));
                    }
                }
                if (PAIR && j == nt - 1) s_fin[0][PAIR ? lrow : 0] = m, s_fin[1][PAIR ? lrow : 0] = l;
                tc::tmem_st_wait();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(smem_u32(&bars.p_full[sb]));
            }
            if (!PAIR && !dead) {
                if (nt == 0 || wait(bars.o_full[rt], nt - 1)) {
                    tc::fence_after_sync();
#pragma unroll
                    for (int c = 0; c < CH; c++) {
                        uint32_t v[32];
                        if (nt > 0) {
                            tc::tmem_ld32(tl + 256 + rt * 128 + c * 32, v);
                            tc::tmem_ld_wait();
                        }
                        float f[32];
#pragma unroll
                        for (int i = 0; i < 32; i++) f[i] = nt > 0 ? __uint_as_float(v[i]) : 0.0f;
                        finish(c, f, l);
                    }
                    put_lse(m, l);
                }
            }
        }
    }
    if (dead && lane == 0) atomicOr(kv.status, (unsigned)DERR_TIMEOUT);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    if (w == 13) tc::tmem_dealloc(tm, 512);
}

template <typename T, int CODE, int D>
static cudaError_t prompt_launch(const KvMaps& maps, const KvArg& kv, const AttendArg& a, cudaStream_t s) {
    using S = PromptShape<D, sizeof(T) == 4>;
    auto k = kv_prompt_kernel<T, CODE, D>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(k, S::SMEM, done);
    if (e != cudaSuccess) return e;
    const int64_t group = a.q.heads / kv.heads, per = 128 * S::NRT;
    // an upper bound of the row tiles: whole ones, and a partial one per request
    const int64_t ctas = ((int64_t)a.T * group / per + min(a.R, a.T)) * kv.heads;
    if (ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
    return launch_pdl(k, dim3((unsigned)ctas), dim3(PT), S::SMEM, s, maps.k, maps.v, kv, a);
}

template <typename T, int CODE>
static cudaError_t prompt_dims(const KvMaps& maps, const KvArg& kv, const AttendArg& a, cudaStream_t s) {
    return kv.dim == 64 ? prompt_launch<T, CODE, 64>(maps, kv, a, s) : prompt_launch<T, CODE, 128>(maps, kv, a, s);
}

cudaError_t launch_prompt(const KvMaps& maps, const KvArg& kv, const AttendArg& a, uint32_t type, int code, cudaStream_t s) {
    const bool i8 = code == RMOE_KV_INT8;
    if (type == T_F32) return i8 ? prompt_dims<float, RMOE_KV_INT8>(maps, kv, a, s) : prompt_dims<float, RMOE_KV_E4M3>(maps, kv, a, s);
    if (type == T_F16) return i8 ? prompt_dims<__half, RMOE_KV_INT8>(maps, kv, a, s) : prompt_dims<__half, RMOE_KV_E4M3>(maps, kv, a, s);
    return i8 ? prompt_dims<__nv_bfloat16, RMOE_KV_INT8>(maps, kv, a, s) : prompt_dims<__nv_bfloat16, RMOE_KV_E4M3>(maps, kv, a, s);
}

}  // namespace rmoe
