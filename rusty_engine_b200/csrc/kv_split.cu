// kv_split.cu -- attention over the 8-bit paged cache for few query rows per request: decoded
// tokens, short speculative chunks.  The work is reading the cache once; it is bound by HBM.
//
// Mathematics.  With x_j = scale log2(e) ks_j q.kc_j + log2(vs_j) over the keys j that a row sees,
//   out = sum_j 2^(x_j - M) vc_j / sum_j 2^(x_j - M) / vs_j ,   lse = (M + log2 of that sum) ln 2
// for any M; M is the running maximum of x_j.  Folding the V scale into the exponent keeps the
// weights of P V in (0, 1] whatever the scales are (v_scale_floor gives their limits).  Codes are exact in
// fp16; q is carried as fp16 times a power of two per row and the weights as fp16 times
// 2^15 (f32 calls: both as pairs, hi + lo), so that a weight has its 11 bits down to 2^-29 of the row's
// largest (f32 calls: 22 bits down to 2^-18, one less for each factor 2 from there).  All sums are f32.
//
// Shape.  A unit of work is a tile of TW tokens of one item (request, kv head, tile of NR rows);
// rows are a request's new tokens x the query heads that share the kv head.  All units of the call
// are numbered, every warp of the grid takes an equal share of consecutive ones, so any mix of
// lengths balances to one tile; no warp waits for another until its share is done.  A warp streams
// its tiles by TMA into its own ring (its own mbarriers, no CTA-wide step) and works with
// mma.sync on the transposed products S^T = K q^T and O^T = V^T P^T: tokens and head elements are
// the M = 16 side, rows the N = 8 side, so eight rows fill the instruction.  The codes widen to
// fp16 in the operand registers; the order of d inside a contraction and of tokens inside a tile
// are free, and are chosen so that each lane's operand is the 16 bytes that it reads.
//
// A tile of keys that none of an item's rows sees (after a causal prompt's early rows, before a
// window) is neither fetched nor computed, and early and late row tiles take turns in the numbering, so
// that the shares stay alike: a prompt of 2048 tokens, 16 heads over 4 of 256, 713 -> 477 us in bf16, 878
// -> 588 in f32.  The bookkeeping costs two requests of 131071 tokens 0.3 us.
//
// Joining.  A share's incomplete first and last items leave (M, l, O) pieces; the CTA joins its
// warps' pieces, and items that span CTAs go through a workspace slot per CTA, where the last
// arriving CTA (an atomic count, nobody waits) joins them in CTA order: the result does not depend
// on timing.
//
// Measured (B200, int8 unless said): 32 requests of 2048 to 8192 tokens, bf16: 41.5 us, 171 MB, 4.1
// TB/s = 63% of the copy rate (f32 47.7); 2 requests of 131071 tokens, fp16, e4m3: 45.7 us, 206 MB, 4.5 TB/s;
// one of 97 tokens, f32: 8.0 us; 512 requests of up to 512 tokens, bf16: 52.9 us, of up to 2048: 128.9.  DRAM traffic is the algorithmic bytes, the issue slots are 41% busy: what is
// above the floor is latency, the steps before the first tile (lengths, block table and the first copy,
// one after the other) and the joining at the end.
#include <algorithm>

#include "kv_attend.h"
#include "kv_widen.cuh"
#include "rope.cuh"
#include "tc_ptx.cuh"

namespace rmoe {

static constexpr int SPLIT_NW = 8;      // warps per CTA
static constexpr int SPLIT_DEPTH = 2;   // tiles in a warp's ring
static constexpr int SPLIT_MAX_SMS = 160;  // CTAs at most

template <int D>
struct SplitShape {
    static constexpr int TW = D == 256 ? 16 : 32;     // tokens per tile
    static constexpr int STAGE = 2 * TW * D;          // K, then V
    static constexpr int MT = TW / 16, KS = D / 16, HF = D / 64;
};

template <int D, int NR>
struct SplitSmem {
    static constexpr int ROW = D + 4;                 // floats between the rows of a piece (bank offset)
    static constexpr int PIECE = NR * (ROW + 2);      // O[NR][ROW], M[NR], l[NR]
    static constexpr int RING = SPLIT_NW * SPLIT_DEPTH * SplitShape<D>::STAGE;
    static constexpr int FIRST = SPLIT_NW * PIECE * 4;
    static constexpr int TOTAL = RING + FIRST + 1024;  // + alignment of the ring
};

// What the warps need of a request.
struct SplitReq {
    int q0, n;       // its first token and its token count
    int pos0;        // position of its first token
    int hi;          // keys 0 .. hi - 1 exist
    int t0, tiles;   // tiles of an item
    int items;       // row tiles x kv heads
};

__device__ __forceinline__ SplitReq split_req(const AttendArg& a, int r, int heads, int group, int bs, int nr, int tw,
                                              int64_t max_rows) {
    SplitReq q;
    const int c0 = __ldg(a.cu + r), c1 = __ldg(a.cu + r + 1), len = __ldg(a.lens + r);
    q.q0 = min(max(c0, 0), a.T);
    q.n = max(0, min(c1, a.T) - q.q0);
    q.pos0 = len - (c1 - c0);
    const int64_t rows = (int64_t)q.n * group;
    q.hi = (int)min((int64_t)max(len, 0), (int64_t)a.max_blocks * bs);
    const int lo = first_seen(a.window, q.pos0);
    q.t0 = min(lo, q.hi) / tw;
    q.tiles = max(1, (q.hi + tw - 1) / tw - q.t0);
    q.items = rows > max_rows ? 0 : (int)((rows + nr - 1) / nr) * heads;
    return q;
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}

// Item -> kv head and tile of rows.  Early and late row tiles take turns: an early row of a causal
// prompt sees few keys, and a warp's share of consecutive items then holds as many of either kind.
struct SplitItem { int kh, rt; };
__device__ __forceinline__ SplitItem split_item(int item, int items, int heads) {
    if (items == heads) return {item, 0};
    const int rts = items / heads, k = item / (2 * heads), j = item - k * 2 * heads;
    if (2 * k + 1 == rts) return {j, k};  // the middle one has no partner
    return {j >> 1, (j & 1) ? rts - 1 - k : k};
}

// Keys that some row of the row tile sees: lo .. hi - 1.
struct SplitKeys { int lo, hi; };
__device__ __forceinline__ SplitKeys split_keys(const AttendArg& a, const SplitReq& q, int rt, int nr, int group) {
    if (q.n == 1) return {0, q.hi};  // a decoded token: its tiles begin and end with its keys
    const int first = rt * nr / group, last = min(q.n - 1, (rt * nr + nr - 1) / group);
    return {first_seen(a.window, q.pos0 + first), min(q.pos0 + last + 1, q.hi)};
}

struct SplitPiece {   // where a piece belongs
    int64_t a;        // the item's first unit
    int tiles;
    int q0, n, row0, head;
    int flags;        // 1: valid, 2: holds the item's first tile, 4: holds its last
};

// a / b for a >= 0, b > 0: in 32 bits where they fit (a 64-bit division is a hundred instructions).
__device__ __forceinline__ int64_t quot(int64_t a, int64_t b) {
    return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

struct SplitStart {   // where a warp's share begins
    SplitReq rq;
    int r;
    int64_t rem;      // units of the request before it
};

template <typename T, int CODE, int D, int NR>
__global__ void __launch_bounds__(SPLIT_NW * 32, 1)
kv_split_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, KvArg kv, AttendArg a,
                SplitWs ws) {
    using S = SplitShape<D>;
    using M = SplitSmem<D, NR>;
    constexpr int NW = SPLIT_NW, NT = NW * 32, DEPTH = SPLIT_DEPTH, TW = S::TW, MT = S::MT, KS = S::KS, HF = S::HF;
    constexpr int QT = NR / 8;                 // n-tiles of 8 rows
    constexpr bool PAIR = sizeof(T) == 4;      // f32: hi + lo
    constexpr bool PRE = !PAIR && NR * D <= 1024;  // q is asked for ahead where registers allow
    constexpr int VB = D == 64 ? 8 : 16;       // V bytes per lane, token and 128-byte box
    constexpr int BX = D == 256 ? 2 : 1;       // 128-byte boxes per row
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t s_full[NW][DEPTH];
    __shared__ __align__(8) float s_scale[NW][DEPTH][2][2];  // per box of the tile: K scale (-1: no such block), V scale
    __shared__ SplitStart s_start[NW];
    __shared__ int64_t s_first[NW];
    __shared__ int64_t s_tot[NW];
    __shared__ SplitPiece s_piece[2 * NW];
    __shared__ int s_last;

    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, c = lane & 3;
    const uint32_t ring0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* ring_ptr = smem_raw + (ring0 - smem_u32(smem_raw));
    const int heads = kv.heads, bs = kv.bs, group = a.group;

    const int br = min(bs, TW), nb = TW / br;  // rows and number of a tile's boxes
    pdl_trigger();
    // the prompt kernel before this one had its inputs when it let this one start, and its requests
    // are not this one's: it is only waited for at the end
    if (!a.prompts) pdl_wait();

    // ---- this warp's share of the units ----
    if (lane < 2) s_piece[2 * w + lane].flags = 0;
    if (lane == 0) {
        for (int i = 0; i < DEPTH; i++) tc::mbar_init(smem_u32(&s_full[w][i]), 1 + nb);
        tc::fence_mbar_init();
    }
    __syncwarp();
    const int bx = blockIdx.x;
    int64_t each = 0, wbase = 0, wlen = 0;  // units of a CTA; this warp's first unit and their number
    int extra = 0;                           // the first `extra` CTAs take one unit more
    auto shares = [&](int64_t W) {
        // a share of less than a tile per warp would only add joining
        const int active = (int)min((int64_t)gridDim.x, (W + NW - 1) / NW);
        each = active ? quot(W, active) : 0;
        extra = (int)(W - each * active);
        const int64_t n = bx < active ? each + (bx < extra) : 0;
        wbase = each * bx + min(bx, extra) + n / NW * w + min(w, (int)(n % NW));
        wlen = n / NW + (w < n % NW);
    };
    auto scan = [&](int64_t x) {  // inclusive, over the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        return x;
    };
    // the request of the warp's first unit, and how many of its units come before
    SplitReq rq{};
    int r = 0;
    int64_t rem = 0, max_rows = INT64_MAX;
    if (a.R <= 32 && !a.prompts) {  // every warp sums up by itself: two barriers less, 1.5 us
        if (lane < a.R) rq = split_req(a, lane, heads, group, bs, NR, TW, max_rows);
        const int64_t mine = (int64_t)rq.items * rq.tiles, incl = scan(mine), at = incl - mine;
        shares(__shfl_sync(0xffffffffu, incl, 31));
        const unsigned own = __ballot_sync(0xffffffffu, wbase >= at && wbase < at + mine);
        r = own ? __ffs(own) - 1 : 0;
        rem = wbase - __shfl_sync(0xffffffffu, at, r);
        int* f = reinterpret_cast<int*>(&rq);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(SplitReq) / 4); i++) f[i] = __shfl_sync(0xffffffffu, f[i], r);
    } else {
        const int per = (a.R + NT - 1) / NT;
        if (a.prompts) max_rows = split_max_rows(a, heads, group, s_tot);
        int64_t mine = 0;
        for (int i = tid * per; i < min(a.R, (tid + 1) * per); i++) {
            rq = split_req(a, i, heads, group, bs, NR, TW, max_rows);
            mine += (int64_t)rq.items * rq.tiles;
        }
        const int64_t incl = scan(mine);
        if (lane == 31) s_tot[w] = incl;
        __syncthreads();
        int64_t before = 0, W = 0;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            if (i < w) before += s_tot[i];
            W += s_tot[i];
        }
        shares(W);
        // the thread that holds a warp's first unit tells it where that is
        if (lane == 0) s_first[w] = wlen > 0 ? wbase : -1;
        __syncthreads();
        const int64_t at = before + incl - mine;
        if (mine > 0)
#pragma unroll 1
            for (int i = 0; i < NW; i++) {
                const int64_t u = s_first[i];
                if (u >= at && u < at + mine) {
                    int64_t left = u - at;
                    int k = tid * per;
                    SplitReq q = rq;
                    if (per > 1) {
                        q = split_req(a, k, heads, group, bs, NR, TW, max_rows);
                        while (left >= (int64_t)q.items * q.tiles) {
                            left -= (int64_t)q.items * q.tiles;
                            q = split_req(a, ++k, heads, group, bs, NR, TW, max_rows);
                        }
                    }
                    s_start[i] = SplitStart{q, k, left};
                }
            }
        __syncthreads();
        if (wlen > 0) {
            rq = s_start[w].rq;
            r = s_start[w].r;
            rem = s_start[w].rem;
        }
    }

    if (wlen > 0) {
        int item = (int)quot(rem, rq.tiles), tile = (int)(rem - (int64_t)item * rq.tiles);

        // the rows of the current item, and its q
        int kh, row0, tok0, rem0;
        uint4 qraw[QT][HF][sizeof(T)];
        // row row0 + i is token tok0 + (rem0 + i) / group, head (rem0 + i) % group of the group
        auto tok_of = [&](int i) { return tok0 + (group == 1 ? i : (int)__umulhi((uint32_t)(rem0 + i), a.group_inv)); };
        auto next_rows = [&]() {
            const SplitItem it = split_item(item, rq.items, heads);
            kh = it.kh;
            row0 = it.rt * NR;
            tok0 = row0 / group;
            rem0 = row0 - tok0 * group;
#pragma unroll
            for (int nt = 0; nt < QT; nt++) {
                const int tok = tok_of(nt * 8 + g), gh = row0 + nt * 8 + g - tok * group;
                const T* qp = reinterpret_cast<const T*>(a.q.p) + (int64_t)(rq.q0 + (tok < rq.n ? tok : 0)) * a.q.st +
                              (int64_t)(kh * group + gh) * a.q.sh;
#pragma unroll
                for (int hf = 0; hf < HF; hf++) {
                    const T* x = qp + (hf * 4 + c) * 16;
                    if (a.q.vec) {
#pragma unroll
                        for (int i = 0; i < (int)sizeof(T); i++) qraw[nt][hf][i] = *(reinterpret_cast<const uint4*>(x) + i);
                    } else {
                        T y[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) y[i] = x[i];
#pragma unroll
                        for (int i = 0; i < (int)sizeof(T); i++) qraw[nt][hf][i] = *(reinterpret_cast<const uint4*>(y) + i);
                    }
                }
            }
        };
        if (PRE) next_rows();

        // ---- the issuing side: runs DEPTH tiles ahead ----
        SplitReq pq = rq;
        int pr = r, pitem = item, ptile = tile;
        int64_t pleft = wlen;
        int pblk = -1;
        SplitItem pit = split_item(pitem, pq.items, heads);
        SplitKeys pkeys = split_keys(a, pq, pit.rt, NR, group);
        auto lookup = [&]() {  // lane b < nb: the block of box b of the tile to issue next
            const int j = (pq.t0 + ptile) * TW + lane * br;
            pblk = -1;
            if (lane < nb && pleft > 0 && j < pq.hi) pblk = __ldg(a.table + (int64_t)pr * a.max_blocks + (j >> kv.shift));
        };
        lookup();
        auto issue = [&](int stage) {
            const uint32_t bar = smem_u32(&s_full[w][stage]);
            const int j = (pq.t0 + ptile) * TW + lane * br;
            // a tile that no row sees is not fetched: its boxes count as missing
            const int j0 = (pq.t0 + ptile) * TW;
            const bool want = lane < nb && j < pq.hi && j0 < pkeys.hi && j0 + TW > pkeys.lo, ok = want && (unsigned)pblk < (unsigned)kv.n_blocks;
            // (a block whose keys all lie before the window may have been given back)
            if (want && !ok && j + br > first_seen(a.window, pq.pos0 + pit.rt * NR / group)) atomicOr(kv.status, (unsigned)DERR_INDEX);
            const unsigned mask = __ballot_sync(0xffffffffu, ok);
            if (lane == 0) tc::mbar_arrive_expect_tx(bar, __popc(mask) * br * D * 2);
            __syncwarp();
            if (ok) {
                const int64_t bh = (int64_t)pblk * heads + pit.kh;
                const int row = (int)(bh * bs + (j & (bs - 1)));
                const uint32_t dst = ring0 + (w * DEPTH + stage) * S::STAGE + lane * br * (D < 128 ? D : 128);
#pragma unroll
                for (int x = 0; x < BX; x++) {
                    tc::tma_2d(dst + x * TW * 128, &kmap, x * 128, row, bar);
                    tc::tma_2d(dst + TW * D + x * TW * 128, &vmap, x * 128, row, bar);
                }
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(smem_u32(&s_scale[w][stage][lane][0])), "l"(kv.ks + bh) : "memory");
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(smem_u32(&s_scale[w][stage][lane][1])), "l"(kv.vs + bh) : "memory");
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(bar) : "memory");
            } else if (lane < nb) {
                s_scale[w][stage][lane][0] = -1.0f;
                s_scale[w][stage][lane][1] = 1.0f;
                tc::mbar_arrive(bar);
            }
            if (--pleft > 0 && ++ptile == pq.tiles) {
                ptile = 0;
                if (++pitem == pq.items) {
                    pitem = 0;
                    do pq = split_req(a, ++pr, heads, group, bs, NR, TW, max_rows);
                    while (pq.items == 0);
                }
                pit = split_item(pitem, pq.items, heads);
                pkeys = split_keys(a, pq, pit.rt, NR, group);
            }
            lookup();
        };
        for (int i = 0; i < DEPTH; i++)
            if (pleft > 0) issue(i);

        // ---- the computing side ----
        // position in a token group of 8 of the S^T row n, and of d chunks over the rows of O^T:
        // the two rows of a quarter-warp's 16-byte reads then fall into different halves of the banks
        const int tg = D == 64 ? g : (g >> 1) + 4 * (g & 1);
        const int t2c = D == 64 ? 2 * c : c, t2c1 = D == 64 ? 2 * c + 1 : c + 4;  // rows 2c and 2c + 1
        const int vg = (g >> 1) + 4 * (g & 1);
        int64_t left = wlen;
        uint32_t cnt = 0;
        bool dead = false, firstseg = true;
        while (left > 0 && !dead) {
            const int seg = (int)min(left, (int64_t)(rq.tiles - tile));
            if (!PRE) next_rows();
            // q rows as B operands, scaled to the fp16 range row by row
            uint32_t qh[QT][KS][2], ql[PAIR ? QT : 1][PAIR ? KS : 1][2];
            float qs[QT][2];
            int vhi[QT][2], vlo[QT][2];
#pragma unroll
            for (int nt = 0; nt < QT; nt++) {
                const bool live = tok_of(nt * 8 + g) < rq.n;
                float v[HF][16], mx = 0.0f;
#pragma unroll
                for (int hf = 0; hf < HF; hf++) {
                    T y[16];
#pragma unroll
                    for (int i = 0; i < (int)sizeof(T); i++) *(reinterpret_cast<uint4*>(y) + i) = qraw[nt][hf][i];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        v[hf][e] = live ? Elt<T>::get(y[e]) : 0.0f;
                        mx = fmaxf(mx, fabsf(v[hf][e]));
                    }
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const int e = q_exponent(mx);
                const float dn = exp2i(-e);
#pragma unroll
                for (int hf = 0; hf < HF; hf++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int p = 0; p < 2; p++) {
                            const float x = v[hf][4 * i + 2 * p] * dn, y = v[hf][4 * i + 2 * p + 1] * dn;
                            const uint32_t hh = pack_f16x2(x, y);
                            qh[nt][hf * 4 + i][p] = hh;
                            if (PAIR) {
                                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hh));
                                ql[nt][hf * 4 + i][p] = pack_f16x2(x - f.x, y - f.y);
                            }
                        }
                const float up = exp2i(e) * a.scale * LOG2E;
#pragma unroll
                for (int i = 0; i < 2; i++) {  // of the rows 2c, 2c + 1 whose sums this lane holds
                    qs[nt][i] = __shfl_sync(0xffffffffu, up, (2 * c + i) * 4);
                    const int t2 = tok_of(nt * 8 + 2 * c + i), p = rq.pos0 + t2;
                    vhi[nt][i] = t2 < rq.n ? min(p + 1, rq.hi) : 0;
                    vlo[nt][i] = first_seen(a.window, p);
                }
            }
            // keys that every row of the tile sees: no masks there
            const int last = min(rq.n - 1, tok_of(NR - 1)), firstt = tok0;
            const int all_hi = min(rq.pos0 + firstt + 1, rq.hi);
            const int all_lo = first_seen(a.window, rq.pos0 + last);
            const int any_lo = first_seen(a.window, rq.pos0 + firstt);
            const int any_hi = min(rq.pos0 + last + 1, rq.hi);

            float o[QT][KS][4], m[QT][2], l[QT][2];
#pragma unroll
            for (int nt = 0; nt < QT; nt++) {
                m[nt][0] = m[nt][1] = -INFINITY;
                l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
                for (int i = 0; i < KS; i++) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
            }
            for (int s = 0; s < seg; s++, cnt++) {
                const int stage = cnt % DEPTH;
                if (!__all_sync(0xffffffffu, tc::mbar_wait_tries(smem_u32(&s_full[w][stage]), (cnt / DEPTH) & 1))) {
                    dead = true;
                    break;
                }
                const uint32_t kb = ring0 + (w * DEPTH + stage) * S::STAGE, vb = kb + TW * D;
                const int j0 = (rq.t0 + tile + s) * TW;
                if (j0 < any_hi && j0 + TW > any_lo) {  // some row sees it; otherwise it was not fetched
                    float kscale[MT], lv[MT], iv[MT];
                    bool gone = false;
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        const float2 sc = *reinterpret_cast<const float2*>(s_scale[w][stage][MT == 2 && br == 16 ? i : 0]);
                        const float vs = v_scale_floor(sc.y);
                        kscale[i] = sc.x;
                        lv[i] = lg2(vs);
                        iv[i] = rcp(vs);
                        gone |= kscale[i] < 0.0f;
                    }
                    const bool masked = gone || j0 < all_lo || j0 + TW > all_hi;
                    if (CODE == RMOE_KV_E4M3 && masked) {
                        // places that no row sees may hold the format's NaN, and 0 * NaN is NaN
                        for (int i = lane; i < TW * (D / 16); i += 32) {
                            const int t = i / (D / 16), ch = i % (D / 16), j = j0 + t;
                            const bool no = j >= rq.hi || j < any_lo || (MT == 2 && t >= 16 ? kscale[MT - 1] : kscale[0]) < 0.0f;
                            // whole rows are cleared, so the swizzle inside a row does not matter
                            if (no)
                                *reinterpret_cast<uint4*>(ring_ptr + (vb - ring0) + (D == 256 ? (ch / 8) * TW * 128 + t * 128 + (ch % 8) * 16 : t * D + ch * 16)) =
                                    make_uint4(0, 0, 0, 0);
                        }
                        tc::fence_proxy_async_smem();  // before the next copy into this stage
                        __syncwarp();
                    }
                    // S^T = K q^T: rows tokens, columns query rows.  The tensor cores cut the sums of a
                    // chain of products short at each step, so a chain is 64 elements long and the
                    // chains are added by the f32 unit (256 elements in one chain cost 1e-5 of the
                    // score); the low halves have their own chain.
                    float st[QT][MT][4], su[PAIR ? QT : 1][PAIR ? MT : 1][4];
#pragma unroll
                    for (int nt = 0; nt < QT; nt++)
#pragma unroll
                        for (int i = 0; i < MT; i++) {
                            st[nt][i][0] = st[nt][i][1] = st[nt][i][2] = st[nt][i][3] = 0.0f;
                            if (PAIR) su[nt][i][0] = su[nt][i][1] = su[nt][i][2] = su[nt][i][3] = 0.0f;
                        }
#pragma unroll
                    for (int hf = 0; hf < HF; hf++)
#pragma unroll
                        for (int i = 0; i < MT; i++) {
                            uint4 x[2];
#pragma unroll
                            for (int z = 0; z < 2; z++) {
                                const int row = 16 * i + 8 * z + tg;
                                x[z] = D == 64 ? lds128(kb + row * 64 + ((c ^ ((row >> 1) & 3)) << 4))
                                               : lds128(kb + (hf / 2) * TW * 128 + row * 128 + ((((hf & 1) * 4 + c) ^ (row & 7)) << 4));
                            }
                            float ch[QT][4];
#pragma unroll
                            for (int nt = 0; nt < QT; nt++) ch[nt][0] = ch[nt][1] = ch[nt][2] = ch[nt][3] = 0.0f;
                            const uint32_t x0[4] = {x[0].x, x[0].y, x[0].z, x[0].w}, x1[4] = {x[1].x, x[1].y, x[1].z, x[1].w};
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                uint32_t f[4];
                                widen4<CODE>(x0[k], f[0], f[2]);
                                widen4<CODE>(x1[k], f[1], f[3]);
#pragma unroll
                                for (int nt = 0; nt < QT; nt++) {
                                    mma_f16_16816(ch[nt], f, qh[nt][hf * 4 + k][0], qh[nt][hf * 4 + k][1]);
                                    if (PAIR) mma_f16_16816(su[nt][i], f, ql[nt][hf * 4 + k][0], ql[nt][hf * 4 + k][1]);
                                }
                            }
#pragma unroll
                            for (int nt = 0; nt < QT; nt++)
#pragma unroll
                                for (int e = 0; e < 4; e++) st[nt][i][e] += ch[nt][e];
                        }
                    // weights
                    uint32_t ph[QT][MT][2], pl[PAIR ? QT : 1][MT][2];
#pragma unroll
                    for (int nt = 0; nt < QT; nt++) {
                        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                        for (int i = 0; i < MT; i++) {
                            const float sc[2] = {qs[nt][0] * kscale[i], qs[nt][1] * kscale[i]};
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                st[nt][i][e] = fmaf(PAIR ? st[nt][i][e] + su[nt][i][e] : st[nt][i][e], sc[e & 1], lv[i]);
                        }
                        if (masked) {
#pragma unroll
                            for (int i = 0; i < MT; i++)
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    const int q = e & 1, j = j0 + 16 * i + 8 * (e >> 1) + tg;
                                    if (j >= vhi[nt][q] || j < vlo[nt][q] || kscale[i] < 0.0f) st[nt][i][e] = -INFINITY;
                                }
                            asm volatile("" ::: "memory");  // a branch: few tiles are masked
                        }
#pragma unroll
                        for (int i = 0; i < MT; i++)
#pragma unroll
                            for (int e = 0; e < 4; e++) mx[e & 1] = fmaxf(mx[e & 1], st[nt][i][e]);
                        float al[2], mu[2];
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            mx[q] = fmaxf(mx[q], __shfl_xor_sync(0xffffffffu, mx[q], 4));
                            mx[q] = fmaxf(mx[q], __shfl_xor_sync(0xffffffffu, mx[q], 8));
                            mx[q] = fmaxf(mx[q], __shfl_xor_sync(0xffffffffu, mx[q], 16));
                            const float mn = fmaxf(m[nt][q], mx[q]);
                            mu[q] = mn == -INFINITY ? 0.0f : mn;
                            al[q] = ex2(m[nt][q] - mu[q]);
                            m[nt][q] = mn;
                        }
                        if (__any_sync(0xffffffffu, al[0] != 1.0f || al[1] != 1.0f)) {
                            l[nt][0] *= al[0];
                            l[nt][1] *= al[1];
#pragma unroll
                            for (int i = 0; i < KS; i++) {
                                o[nt][i][0] *= al[0];
                                o[nt][i][1] *= al[1];
                                o[nt][i][2] *= al[0];
                                o[nt][i][3] *= al[1];
                            }
                        }
#pragma unroll
                        for (int i = 0; i < MT; i++) {
                            float p[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                p[e] = ex2(st[nt][i][e] - mu[e & 1]);
                                l[nt][e & 1] = fmaf(p[e], iv[i], l[nt][e & 1]);
                            }
#pragma unroll
                            for (int z = 0; z < 2; z++) {
                                const float x = p[2 * z] * W_UP, y = p[2 * z + 1] * W_UP;
                                const uint32_t hh = pack_f16x2(x, y);
                                ph[nt][i][z] = movmatrix(hh);
                                if (PAIR) {
                                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hh));
                                    pl[nt][i][z] = movmatrix(pack_f16x2(x - f.x, y - f.y));
                                }
                            }
                        }
                    }
                    // O^T += V^T P^T: rows head elements, columns query rows
#pragma unroll
                    for (int i = 0; i < MT; i++)
#pragma unroll
                        for (int x = 0; x < BX; x++) {
                            uint32_t v[4][VB / 4];
#pragma unroll
                            for (int z = 0; z < 4; z++) {
                                const int row = 16 * i + 8 * (z >> 1) + ((z & 1) ? t2c1 : t2c);
                                if (D == 64) {
                                    const uint2 y = lds64(vb + row * 64 + (((vg >> 1) ^ ((row >> 1) & 3)) << 4) + (vg & 1) * 8);
                                    v[z][0] = y.x;
                                    v[z][1] = y.y;
                                } else {
                                    const uint4 y = lds128(vb + x * TW * 128 + row * 128 + ((vg ^ (row & 7)) << 4));
                                    v[z][0] = y.x;
                                    v[z][1] = y.y;
                                    v[z][VB / 4 - 2] = y.z;
                                    v[z][VB / 4 - 1] = y.w;
                                }
                            }
#pragma unroll
                            for (int k = 0; k < VB / 4; k++) {
                                uint32_t f[2][4];  // of the two O^T tiles of this word
                                widen4<CODE>(__byte_perm(v[0][k], v[1][k], 0x5140), f[0][0], f[0][1]);
                                widen4<CODE>(__byte_perm(v[2][k], v[3][k], 0x5140), f[0][2], f[0][3]);
                                widen4<CODE>(__byte_perm(v[0][k], v[1][k], 0x7362), f[1][0], f[1][1]);
                                widen4<CODE>(__byte_perm(v[2][k], v[3][k], 0x7362), f[1][2], f[1][3]);
#pragma unroll
                                for (int nt = 0; nt < QT; nt++)
#pragma unroll
                                    for (int y = 0; y < 2; y++) {
                                        float* acc = o[nt][x * 8 + 2 * k + y];
                                        if (PAIR) {  // a chain of two, as above
                                            float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                            mma_f16_16816(t, f[y], pl[nt][i][0], pl[nt][i][1]);
                                            mma_f16_16816(t, f[y], ph[nt][i][0], ph[nt][i][1]);
#pragma unroll
                                            for (int e = 0; e < 4; e++) acc[e] += t[e];
                                        } else {
                                            mma_f16_16816(acc, f[y], ph[nt][i][0], ph[nt][i][1]);
                                        }
                                    }
                            }
                        }
                }
                __syncwarp();  // every lane has read the stage
                if (pleft > 0) issue(stage);
            }
            if (dead) break;
            // ---- the item's share is done ----
#pragma unroll
            for (int nt = 0; nt < QT; nt++)
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    l[nt][q] += __shfl_xor_sync(0xffffffffu, l[nt][q], 4);
                    l[nt][q] += __shfl_xor_sync(0xffffffffu, l[nt][q], 8);
                    l[nt][q] += __shfl_xor_sync(0xffffffffu, l[nt][q], 16);
                }
            const bool starts = tile == 0, ends = tile + seg == rq.tiles;
            if (starts && ends) {
#pragma unroll
                for (int nt = 0; nt < QT; nt++)
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        const int tok = tok_of(nt * 8 + 2 * c + q);
                        if (tok >= rq.n) continue;
                        const int h = kh * group + row0 + nt * 8 + 2 * c + q - tok * group;
                        const float inv = l[nt][q] > 0.0f ? W_DOWN / l[nt][q] : (l[nt][q] == 0.0f ? 0.0f : l[nt][q]);
                        T* op = reinterpret_cast<T*>(a.out.p) + (int64_t)(rq.q0 + tok) * a.out.st + h * a.out.sh;
#pragma unroll
                        for (int x = 0; x < BX; x++)
#pragma unroll
                            for (int b = 0; b < VB / 8; b++) {
                                float v[8];
#pragma unroll
                                for (int e = 0; e < 8; e++) v[e] = o[nt][x * 8 + b * 4 + e / 2][(e & 1) * 2 + q] * inv;
                                store8(op + x * 128 + vg * VB + b * 8, a.out.vec, v);
                            }
                        if (g == 0 && a.lse)
                            a.lse[(int64_t)(rq.q0 + tok) * a.q.heads + h] =
                                l[nt][q] == 0.0f ? -INFINITY : (m[nt][q] + log2f(l[nt][q])) * LN2;
                    }
            } else {
                const bool into_first = firstseg && left > seg;  // the ring is still in use then
                float* pc = into_first ? reinterpret_cast<float*>(ring_ptr + M::RING) + w * M::PIECE
                                       : reinterpret_cast<float*>(ring_ptr + w * DEPTH * S::STAGE);
#pragma unroll
                for (int nt = 0; nt < QT; nt++)
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        const int row = nt * 8 + 2 * c + q;
                        if (g == 0) pc[NR * M::ROW + row] = m[nt][q], pc[NR * (M::ROW + 1) + row] = l[nt][q];
#pragma unroll
                        for (int x = 0; x < BX; x++)
#pragma unroll
                            for (int e = 0; e < VB; e += 4)
                                *reinterpret_cast<float4*>(pc + row * M::ROW + x * 128 + vg * VB + e) =
                                    make_float4(o[nt][x * 8 + e / 2][q], o[nt][x * 8 + e / 2][2 + q], o[nt][x * 8 + e / 2 + 1][q],
                                                o[nt][x * 8 + e / 2 + 1][2 + q]);
                    }
                if (lane == 0)
                    s_piece[2 * w + (into_first ? 0 : 1)] =
                        SplitPiece{wbase + wlen - left - tile, rq.tiles, rq.q0, rq.n, row0, kh, 1 | (starts ? 2 : 0) | (ends ? 4 : 0)};
            }
            firstseg = false;
            left -= seg;
            tile += seg;
            if (left > 0 && tile == rq.tiles) {
                tile = 0;
                if (++item == rq.items) {
                    item = 0;
                    do rq = split_req(a, ++r, heads, group, bs, NR, TW, max_rows);
                    while (rq.items == 0);
                }
                if (PRE) next_rows();
            }
        }
        if (dead) {  // a copy did not arrive: say so, and let what is in flight land
            if (lane == 0) atomicOr(kv.status, (unsigned)DERR_TIMEOUT);
            for (int64_t k = wlen - pleft; (int64_t)cnt < k; cnt++)
                tc::mbar_wait_tries(smem_u32(&s_full[w][cnt % DEPTH]), (cnt / DEPTH) & 1);
        }
    }

    // ---- tokens of no request ----
    {
        const int first = min(max(__ldg(a.cu), 0), a.T), end = min(max(__ldg(a.cu + a.R), first), a.T);
        const int64_t rest = (int64_t)(a.T - (end - first)) * a.q.heads;
        for (int64_t i = (int64_t)bx * NW + w; i < rest; i += (int64_t)gridDim.x * NW) {
            const int k = (int)(i / a.q.heads), h = (int)(i % a.q.heads), t = k < first ? k : end + (k - first);
            T* o = reinterpret_cast<T*>(a.out.p) + t * a.out.st + h * a.out.sh;
            for (int d = lane; d < D; d += 32) o[d] = Elt<T>::put(0.0f);
            if (lane == 0 && a.lse) a.lse[(int64_t)t * a.q.heads + h] = -INFINITY;
        }
    }

    // ---- joining ----
    __syncthreads();
    auto piece = [&](int i) {
        return (i & 1) ? reinterpret_cast<float*>(ring_ptr + (i >> 1) * DEPTH * S::STAGE)
                       : reinterpret_cast<float*>(ring_ptr + M::RING) + (i >> 1) * M::PIECE;
    };
    // A warp joins a row: lanes hold the pieces' M and l first, then D / 32 neighbouring elements each.
    constexpr int VE = D / 32;
    auto emit = [&](const SplitPiece& pc, int row, float m, float l, const float* o) {
        const int rr = pc.row0 + row, tok = rr / group;
        if (tok >= pc.n) return;
        const int h = pc.head * group + rr - tok * group;
        const float inv = l > 0.0f ? W_DOWN / l : (l == 0.0f ? 0.0f : l);
        T* op = reinterpret_cast<T*>(a.out.p) + (int64_t)(pc.q0 + tok) * a.out.st + (int64_t)h * a.out.sh + lane * VE;
        T y[VE];
#pragma unroll
        for (int i = 0; i < VE; i++) y[i] = Elt<T>::put(o[i] * inv);
        if (a.out.vec) {
            constexpr int B = VE * (int)sizeof(T);  // 4 to 32 bytes
#pragma unroll
            for (int i = 0; i < (B + 15) / 16; i++)
                if (B >= 16) *(reinterpret_cast<uint4*>(op) + i) = *(reinterpret_cast<const uint4*>(y) + i);
                else if (B == 8) *reinterpret_cast<uint2*>(op) = *reinterpret_cast<const uint2*>(y);
                else *reinterpret_cast<uint32_t*>(op) = *reinterpret_cast<const uint32_t*>(y);
        } else {
#pragma unroll
            for (int i = 0; i < VE; i++) op[i] = y[i];
        }
        if (lane == 0 && a.lse)
            a.lse[(int64_t)(pc.q0 + tok) * a.q.heads + h] = l == 0.0f ? -INFINITY : (m + lg2(l)) * LN2;
    };
    auto vec = [&](const float* p, float* v) {  // VE floats
        if (VE == 2) *reinterpret_cast<float2*>(v) = __ldcg(reinterpret_cast<const float2*>(p));
        else
#pragma unroll
            for (int i = 0; i < VE / 4; i++) *(reinterpret_cast<float4*>(v) + i) = __ldcg(reinterpret_cast<const float4*>(p) + i);
    };
    auto wmax = [&](float x) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
        return x;
    };
    auto wsum = [&](float x) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        return x;
    };
    const unsigned valid = __ballot_sync(0xffffffffu, lane < 2 * NW && (s_piece[lane & (2 * NW - 1)].flags & 1));
    for (unsigned todo = valid; todo;) {
        const SplitPiece& pc = s_piece[__ffs(todo) - 1];
        // the slots that hold pieces of this item
        const SplitPiece& mp = s_piece[lane & (2 * NW - 1)];
        const unsigned set = __ballot_sync(0xffffffffu, (todo >> lane & 1) && mp.a == pc.a);
        const bool in = set >> lane & 1;
        const int flags = __reduce_or_sync(0xffffffffu, in ? mp.flags : 0);
        todo &= ~set;
        const bool whole = (flags & 6) == 6;
        float* slot = ws.part + (size_t)(2 * bx + ((flags & 2) ? 1 : 0)) * M::PIECE;
#pragma unroll 1
        for (int row = w; row < NR; row += NW) {
            const float* mine_p = in ? piece(lane) : piece(0);
            const float pm = in ? mine_p[NR * M::ROW + row] : -INFINITY, mm = wmax(pm), mu = mm == -INFINITY ? 0.0f : mm;
            const float f = ex2(pm - mu), ll = wsum(in ? mine_p[NR * (M::ROW + 1) + row] * f : 0.0f);
            float o[VE];
#pragma unroll
            for (int i = 0; i < VE; i++) o[i] = 0.0f;
            for (unsigned rest = set; rest; rest &= rest - 1) {
                const int k = __ffs(rest) - 1;
                const float fk = __shfl_sync(0xffffffffu, f, k);
                const float* p = piece(k) + row * M::ROW + lane * VE;
#pragma unroll
                for (int i = 0; i < VE; i++) o[i] = fmaf(p[i], fk, o[i]);
            }
            if (whole) {
                emit(pc, row, mm, ll, o);
            } else {
#pragma unroll
                for (int i = 0; i < VE; i += 2) __stcg(reinterpret_cast<float2*>(slot + row * M::ROW + lane * VE + i), make_float2(o[i], o[i + 1]));
                if (lane == 0) __stcg(slot + NR * M::ROW + row, mm), __stcg(slot + NR * (M::ROW + 1) + row, ll);
            }
        }
        if (whole) continue;
        // the CTAs that hold the item's first and last unit
        auto cta_of = [&](int64_t u) {
            const int64_t big = extra * (each + 1);
            return (int)(u < big ? quot(u, each + 1) : extra + quot(u - big, each));
        };
        const int c0 = cta_of(pc.a), n = cta_of(pc.a + pc.tiles - 1) - c0 + 1;
        __threadfence();
        __syncthreads();
        if (tid == 0) s_last = atomicAdd(ws.ticket + c0, 1u) == (unsigned)(n - 1);
        __syncthreads();
        if (s_last) {
            __threadfence();
            auto part = [&](int k) { return ws.part + (size_t)(2 * (c0 + k) + (k == 0 ? 1 : 0)) * M::PIECE; };
#pragma unroll 1
            for (int row = w; row < NR; row += NW) {
                float mm = -INFINITY;
                for (int k = lane; k < n; k += 32) mm = fmaxf(mm, __ldcg(part(k) + NR * M::ROW + row));
                mm = wmax(mm);
                const float mu = mm == -INFINITY ? 0.0f : mm;
                float o[VE], ll = 0.0f;
#pragma unroll
                for (int i = 0; i < VE; i++) o[i] = 0.0f;
                for (int k0 = 0; k0 < n; k0 += 32) {
                    const int k1 = min(32, n - k0);
                    const float* mine_p = part(k0 + min(lane, k1 - 1));
                    const float f = lane < k1 ? ex2(__ldcg(mine_p + NR * M::ROW + row) - mu) : 0.0f;
                    ll = fmaf(__ldcg(mine_p + NR * (M::ROW + 1) + row), f, ll);
#pragma unroll 4
                    for (int k = 0; k < k1; k++) {
                        float v[VE];
                        vec(part(k0 + k) + row * M::ROW + lane * VE, v);
                        const float fk = __shfl_sync(0xffffffffu, f, k);
#pragma unroll
                        for (int i = 0; i < VE; i++) o[i] = fmaf(v[i], fk, o[i]);
                    }
                }
                ll = wsum(ll);
                emit(pc, row, mm, ll, o);
            }
            if (tid == 0) ws.ticket[c0] = 0;
        }
        __syncthreads();  // s_last is used again
    }
    if (a.prompts) pdl_wait();
}

template <typename T, int CODE, int D, int NR>
static cudaError_t split_launch(const KvMaps& maps, const KvArg& kv, const AttendArg& a, const SplitWs& ws, int sms, cudaStream_t s) {
    constexpr int smem = SplitSmem<D, NR>::TOTAL;
    static_assert(SplitSmem<D, NR>::PIECE * 4 <= SPLIT_DEPTH * SplitShape<D>::STAGE, "a last piece takes the place of the ring");
    auto k = kv_split_kernel<T, CODE, D, NR>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(k, smem, done);
    if (e != cudaSuccess) return e;
    return launch_pdl(k, dim3(std::min(sms, SPLIT_MAX_SMS)), dim3(SPLIT_NW * 32), smem, s, maps.k, maps.v, kv, a, ws);
}

// nr: 8 or 16 rows per item (16 only up to head_dim 128: the accumulators of 256 alone would take 128
// registers a thread; 8 rows of it spill 44 bytes in f32)
template <typename T, int CODE>
static cudaError_t split_dims(const KvMaps& maps, const KvArg& kv, const AttendArg& a, const SplitWs& ws, int sms, int nr,
                              cudaStream_t s) {
    if (kv.dim == 64)
        return nr == 8 ? split_launch<T, CODE, 64, 8>(maps, kv, a, ws, sms, s) : split_launch<T, CODE, 64, 16>(maps, kv, a, ws, sms, s);
    if (kv.dim == 128)
        return nr == 8 ? split_launch<T, CODE, 128, 8>(maps, kv, a, ws, sms, s) : split_launch<T, CODE, 128, 16>(maps, kv, a, ws, sms, s);
    return split_launch<T, CODE, 256, 8>(maps, kv, a, ws, sms, s);
}

int split_tile_tokens(int dim) { return dim == 256 ? SplitShape<256>::TW : SplitShape<128>::TW; }
size_t split_part_bytes(int dim) { return (size_t)(dim == 256 ? 8 : 16) * (dim + 4 + 2) * 4 * 2; }

cudaError_t launch_split(const KvMaps& maps, const KvArg& kv, const AttendArg& a, const SplitWs& ws, int sms, int nr,
                         uint32_t type, int code, cudaStream_t s) {
    const bool i8 = code == RMOE_KV_INT8;
    if (type == T_F32)
        return i8 ? split_dims<float, RMOE_KV_INT8>(maps, kv, a, ws, sms, nr, s) : split_dims<float, RMOE_KV_E4M3>(maps, kv, a, ws, sms, nr, s);
    if (type == T_F16)
        return i8 ? split_dims<__half, RMOE_KV_INT8>(maps, kv, a, ws, sms, nr, s)
                  : split_dims<__half, RMOE_KV_E4M3>(maps, kv, a, ws, sms, nr, s);
    return i8 ? split_dims<__nv_bfloat16, RMOE_KV_INT8>(maps, kv, a, ws, sms, nr, s)
              : split_dims<__nv_bfloat16, RMOE_KV_E4M3>(maps, kv, a, ws, sms, nr, s);
}

}  // namespace rmoe
