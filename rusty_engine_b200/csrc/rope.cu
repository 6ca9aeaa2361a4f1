// rope.cu -- rotary positions: the table of cosines and sines, and turning q and k by it.
//
// Pair i of a head is turned by pos * f_i.  At position 1e5 an f32 product carries an error of
// several milliradians, so the angles are formed in 64 bits, once, when the handle is made, and
// cos and sin are rounded to f32 there; a call reads 4 * rot_dim bytes of table per token against
// (q heads + k heads) * head_dim elements of data (3% more traffic at 36 heads of 128 in bf16).
#include <math.h>

#include <vector>

#include <algorithm>

#include "rope.cuh"
#include "tc_ptx.cuh"

namespace rmoe {

__global__ void __launch_bounds__(256) rope_table_kernel(float2* table, const double* freq, int pairs, uint64_t n,
                                                         double m) {
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) {
        double s, c;
        sincos((double)(i / pairs) * freq[i % pairs], &s, &c);
        table[i] = make_float2((float)(c * m), (float)(s * m));
    }
}

// Units of 16 elements (rope.cuh), spread over all threads: short batches, and heads that do not lie
// one after the other.  16 tokens of 32 + 4 heads of 128 in f32: 2.0 us (B200, calls in a graph), latency.
template <typename T>
__global__ void __launch_bounds__(256, 3) rope_units_kernel(Rows q, Rows qo, Rows k, Rows ko, RopeArg ra, int T_, int dim,
                                                            unsigned* status) {
    pdl_wait();
    pdl_trigger();
    turn_items<T>(q, qo, k, ko, ra, T_, dim, blockIdx.x * 256ll + threadIdx.x, gridDim.x * 256ll, status);
}

// Long batches of heads that lie one after the other: a warp brings a token's q, k and angles into
// its own part of shared memory as bulk copies, turns them there and sends them back as bulk
// copies, three tokens deep.  The copies keep the memory busy with hardly any registers, where
// per-thread loads of 16-bit heads reached 62-70% of the copy rate whatever their number; a ring shared by
// the CTA's warps, in step from token to token, was no faster than those (8192 tokens of 32 + 4 heads of
// 128 in bf16, B200).  A ring per warp: 27.4 us, 153 MB, 5.6 TB/s = 85% of the copy rate;
// 67 MB of q in and out: 25.6 us where a copy takes 24.7.
struct RopeStream {
    uint32_t qb, kb, ab, stage;  // bytes of a token's q, k and angles, and of a stage
    int warps;
};
static constexpr int RS_STAGES = 3, RS_MAX_WARPS = 8;

template <typename T>
__global__ void __launch_bounds__(RS_MAX_WARPS * 32)
    rope_stream_kernel(Rows q, Rows qo, Rows k, Rows ko, RopeArg ra, int T_, int dim, RopeStream rs, unsigned* status) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t s_full[RS_MAX_WARPS][RS_STAGES];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const uint32_t skew = (128u - (smem_u32(smem_raw) & 127u)) & 127u;
    uint8_t* ring = smem_raw + skew + w * RS_STAGES * rs.stage;
    const uint32_t ring_s = smem_u32(ring);
    if (lane == 0) {
        for (int i = 0; i < RS_STAGES; i++) tc::mbar_init(smem_u32(&s_full[w][i]), 1);
        tc::fence_mbar_init();
    }
    __syncwarp();
    pdl_wait();
    pdl_trigger();
    const int step = gridDim.x * rs.warps, t0 = blockIdx.x + w * gridDim.x;  // tokens t0, t0 + step, ...
    const int n = t0 < T_ ? (T_ - 1 - t0) / step + 1 : 0;
    int pos = 0;         // lane l: of token 32 * (i / 32) + l
    unsigned turned = 0; // bit s: the token in stage s is turned
    auto load = [&](int i) {
        const int64_t t = t0 + (int64_t)i * step;
        if ((i & 31) == 0) {
            const int64_t tl = t + (int64_t)lane * step;
            pos = tl < T_ ? __ldg(ra.pos + tl) : 0;
        }
        const int p = __shfl_sync(0xffffffffu, pos, i & 31), s = i % RS_STAGES;
        const bool in = (unsigned)p < (unsigned)ra.max_pos;
        turned = in ? turned | 1u << s : turned & ~(1u << s);
        if (lane == 0) {
            const uint32_t bar = smem_u32(&s_full[w][s]), dst = ring_s + s * rs.stage;
            if (!in) atomicOr(status, (unsigned)DERR_INDEX);
            tc::mbar_arrive_expect_tx(bar, rs.qb + rs.kb + (in ? rs.ab : 0));
            tc::bulk_g2s(dst, q.p + t * q.st * (int64_t)sizeof(T), rs.qb, bar);
            if (rs.kb) tc::bulk_g2s(dst + rs.qb, k.p + t * k.st * (int64_t)sizeof(T), rs.kb, bar);
            if (in) tc::bulk_g2s(dst + rs.qb + rs.kb, ra.table + (int64_t)p * (ra.rot / 2), rs.ab, bar);
        }
    };
    int loaded = 0, i = 0;
    bool dead = false;
    for (; loaded < min(n, RS_STAGES); loaded++) load(loaded);
    const int units = ra.rot >> 4, all = (q.heads + k.heads) * units;  // rotated units only
    for (; i < n; i++) {
        const int s = i % RS_STAGES;
        dead = !__all_sync(0xffffffffu, tc::mbar_wait_tries(smem_u32(&s_full[w][s]), (i / RS_STAGES) & 1));
        if (dead) break;
        uint8_t* st = ring + s * rs.stage;
        const float4* ang = reinterpret_cast<const float4*>(st + rs.qb + rs.kb);
        if (turned >> s & 1) {
            // where a head's units divide the warp, a lane has the same unit of every head and reads
            // its angles once (read per head, their bank conflicts bound the kernel: 32 -> 25 us)
            const bool fixed = (32 % units) == 0;
            float4 cs[4];
            if (fixed)
#pragma unroll
                for (int j = 0; j < 4; j++) cs[j] = ang[lane % units * 4 + j];
            const int hstep = fixed ? 32 / units : 0;
            int h = lane / units, c = lane - h * units;  // k's heads follow q's
#pragma unroll 2
            for (int u = lane; u < all; u += 32) {
                if (!fixed) {
                    h = u / units;
                    c = u - h * units;
#pragma unroll
                    for (int j = 0; j < 4; j++) cs[j] = ang[c * 4 + j];
                }
                int a, b;
                unit_chunks(c, ra.rot, ra.half, a, b);
                T* x = reinterpret_cast<T*>(st) + h * dim;
                float v[16];
                load8(x + a, true, v);
                load8(x + b, true, v + 8);
                turn_unit_by(v, cs, ra.half, ra.sign);
                store8(x + a, true, v);
                store8(x + b, true, v + 8);
                h += hstep;
            }
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            const int64_t t = t0 + (int64_t)i * step;
            const uint32_t src = ring_s + s * rs.stage;
            tc::bulk_s2g(qo.p + t * qo.st * (int64_t)sizeof(T), src, rs.qb);
            if (rs.kb) tc::bulk_s2g(ko.p + t * ko.st * (int64_t)sizeof(T), src + rs.qb, rs.kb);
            tc::bulk_commit();
            tc::bulk_wait_read<1>();  // the token before has left its stage
        }
        __syncwarp();
        if (i > 0 && loaded < n) load(loaded), loaded++;
    }
    if (dead) {
        if (lane == 0) atomicOr(status, (unsigned)DERR_TIMEOUT);
        for (; i < loaded; i++) tc::mbar_wait_tries(smem_u32(&s_full[w][i % RS_STAGES]), (i / RS_STAGES) & 1);
    }
    if (lane == 0) tc::bulk_wait<0>();
}

// Head and rotary sizes that are not multiples of 16: one thread per pair, then per copied element.
template <typename T>
__global__ void __launch_bounds__(256) rope_pairs_kernel(Rows q, Rows qo, Rows k, Rows ko, RopeArg ra, int T_, int dim,
                                                         unsigned* status) {
    pdl_wait();
    pdl_trigger();
    const int per_head = ra.rot / 2 + (dim - ra.rot), per_tok = (q.heads + k.heads) * per_head;
    const uint64_t n = (uint64_t)T_ * per_tok;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) {
        const int t = (int)(i / per_tok), r = (int)(i - (uint64_t)t * per_tok), h = r / per_head, u = r - h * per_head;
        const bool isq = h < q.heads;
        const Rows& in = isq ? q : k;
        const Rows& out = isq ? qo : ko;
        const int hh = isq ? h : h - q.heads;
        const T* x = reinterpret_cast<const T*>(in.p) + t * in.st + hh * in.sh;
        T* y = reinterpret_cast<T*>(out.p) + t * out.st + hh * out.sh;
        if (u >= ra.rot / 2) {
            const int e = u + ra.rot / 2;
            y[e] = x[e];
            continue;
        }
        const int a = ra.half ? u : 2 * u, b = ra.half ? u + ra.rot / 2 : 2 * u + 1;
        float x0 = Elt<T>::get(x[a]), x1 = Elt<T>::get(x[b]);
        const int p = __ldg(ra.pos + t);
        if ((unsigned)p < (unsigned)ra.max_pos) {
            const float2 cs = __ldg(ra.table + (size_t)p * (ra.rot / 2) + u);
            turn(x0, x1, cs.x, ra.sign * cs.y);
        } else if (u == 0 && h == 0) {
            atomicOr(status, (unsigned)DERR_INDEX);
        }
        y[a] = Elt<T>::put(x0);
        y[b] = Elt<T>::put(x1);
    }
}

template <typename T>
static cudaError_t rope_launch(const Rows& q, const Rows& qo, const Rows& k, const Rows& ko, const RopeArg& ra, int T_,
                               int dim, unsigned* status, cudaStream_t s) {
    const bool units = dim % 16 == 0 && ra.rot % 16 == 0;
    const bool rows = q.vec && qo.vec && q.sh == dim && qo.sh == dim && (!k.heads || (k.vec && ko.vec && k.sh == dim && ko.sh == dim));
    // The ring pays for long batches of 16-bit heads, where the stages of three warps fit an SM.  Ring / units in
    // us (B200, heads of 128): 8192 tokens in bf16, 32 + 4 heads 27.0 / 35.4, 64 + 4 53.9 / 63.9, 8 + 2
    // 13.1 / 11.5; 2048 tokens of 32 + 4 9.0 / 10.7; 1184 8.0 / 6.6.  In f32, where a thread has twice the bytes
    // in flight, the units reach 92 to 97% of the copy rate: 8192 tokens of 32 + 4 54.1 / 50.4, 44 + 2 71.9 /
    // 64.7, 8 + 2 15.1 / 16.3; 2048 of 32 + 4 14.4 / 15.1.
    if (units && rows && q.heads && T_ >= 148 * 8) {
        RopeStream rs;
        rs.qb = (uint32_t)(q.heads * dim * sizeof(T));
        rs.kb = (uint32_t)(k.heads * dim * sizeof(T));
        rs.ab = (uint32_t)(ra.rot / 2 * sizeof(float2));
        rs.stage = (rs.qb + rs.kb + rs.ab + 127) / 128 * 128;
        constexpr uint32_t room = 220 << 10;
        rs.warps = (int)std::min<uint32_t>(RS_MAX_WARPS, room / (RS_STAGES * rs.stage));
        if (rs.warps >= 3) {
            static std::atomic<uint64_t> done{0};
            cudaError_t e = allow_smem(rope_stream_kernel<T>, room + 128, done);
            if (e != cudaSuccess) return e;
            return launch_pdl(rope_stream_kernel<T>, dim3(148), dim3(rs.warps * 32), rs.warps * RS_STAGES * rs.stage + 128, s, q, qo, k,
                              ko, ra, T_, dim, rs, status);
        }
    }
    const uint64_t n = (uint64_t)T_ * (q.heads + k.heads) * (units ? dim / 16 : dim - ra.rot / 2), ctas = (n + 255) / 256;
    const unsigned most = units ? 148 * 3 : 148 * 64;  // units: the CTAs that are resident, each thread walks over many
    return launch_pdl(units ? rope_units_kernel<T> : rope_pairs_kernel<T>, dim3((unsigned)(ctas < most ? ctas : most)), dim3(256), 0,
                      s, q, qo, k, ko, ra, T_, dim, status);
}

// Every rope kernel lets the next kernel start only once its own inputs are there (the wait comes
// before the trigger): one that does not read the turned heads need not wait for them.
cudaError_t launch_rope_apply(const Rows& q, const Rows& qo, const Rows& k, const Rows& ko, const RopeArg& ra, int T,
                              int dim, uint32_t type, unsigned* status, cudaStream_t s) {
    if (type == T_F32) return rope_launch<float>(q, qo, k, ko, ra, T, dim, status, s);
    if (type == T_F16) return rope_launch<__half>(q, qo, k, ko, ra, T, dim, status, s);
    return rope_launch<__nv_bfloat16>(q, qo, k, ko, ra, T, dim, status, s);
}

rmoe_status check_rows(const rmoe_rows& a, uint32_t T, uint32_t type, const char* what, Rows& r) {
    const uint32_t es = elt_size(type);
    if (a.heads > 65535) return fail(RMOE_ERR_UNSUPPORTED, "%s: %u heads", what, a.heads);
    if (a.heads && T && !a.data) return fail(RMOE_ERR_INVALID, "%s: null data", what);
    if (reinterpret_cast<uintptr_t>(a.data) % es) return fail(RMOE_ERR_INVALID, "%s: misaligned data", what);
    r.p = static_cast<char*>(a.data);
    r.st = a.stride_t;
    r.sh = a.stride_h;
    r.heads = (int)a.heads;
    r.vec = reinterpret_cast<uintptr_t>(a.data) % 16 == 0 && (a.stride_t * es) % 16 == 0 && (a.stride_h * es) % 16 == 0;
    return RMOE_OK;
}

}  // namespace rmoe

using namespace rmoe;

extern "C" {

rmoe_status rmoe_rope_create(const rmoe_rope_desc* d, rmoe_rope** out) {
    if (!out) return fail(RMOE_ERR_INVALID, "null output handle");
    *out = nullptr;
    if (!d) return fail(RMOE_ERR_INVALID, "null rope description");
    if (d->rot_dim < 2 || d->rot_dim % 2 || d->rot_dim > 4096)
        return fail(RMOE_ERR_INVALID, "rot_dim %u must be even, 2 .. 4096", d->rot_dim);
    if (d->layout > RMOE_ROPE_HALF) return fail(RMOE_ERR_INVALID, "rope layout %u", d->layout);
    if (d->scaling > RMOE_ROPE_YARN) return fail(RMOE_ERR_INVALID, "rope scaling %u", d->scaling);
    if (d->max_pos == 0 || d->max_pos > 0x7fffffffu) return fail(RMOE_ERR_INVALID, "max_pos %u", d->max_pos);
    if (!(d->base > 0.0) || !isfinite(d->base)) return fail(RMOE_ERR_INVALID, "rope base %g", d->base);
    const bool scaled = d->scaling != RMOE_ROPE_PLAIN;
    if (scaled && (!(d->factor >= 1.0) || !isfinite(d->factor)))
        return fail(RMOE_ERR_INVALID, "rope scaling factor %g must be at least 1", d->factor);
    if (d->scaling == RMOE_ROPE_YARN && (d->orig_ctx == 0 || d->base == 1.0))
        return fail(RMOE_ERR_INVALID, "YaRN needs orig_ctx > 0 and a base other than 1");
    const double fast = d->beta_fast == 0.0 ? 32.0 : d->beta_fast, slow = d->beta_slow == 0.0 ? 1.0 : d->beta_slow;
    if (d->scaling == RMOE_ROPE_YARN && (!(fast > 0.0) || !(slow > 0.0) || !(fast >= slow)))
        return fail(RMOE_ERR_INVALID, "YaRN beta_fast %g, beta_slow %g", fast, slow);
    if (!isfinite(d->mscale)) return fail(RMOE_ERR_INVALID, "rope mscale %g", d->mscale);
    const uint32_t pairs = d->rot_dim / 2;
    for (uint32_t i = 0; d->freq_factors && i < pairs; i++)
        if (!(fabsf(d->freq_factors[i]) > 0.0f) || !isfinite(d->freq_factors[i]))
            return fail(RMOE_ERR_INVALID, "freq_factors[%u] = %g", i, d->freq_factors[i]);
    double low = 0, high = 0, m = 1.0;
    if (d->scaling == RMOE_ROPE_YARN) {
        // the pair that makes n turns in orig_ctx positions: base^(-2i/rot) = 2 pi n / orig_ctx
        const double two_pi = 6.283185307179586476925286766559;
        auto at = [&](double n) { return d->rot_dim * log(d->orig_ctx / (n * two_pi)) / (2.0 * log(d->base)); };
        low = fmax(floor(at(fast)), 0.0);
        high = fmin(ceil(at(slow)), (double)d->rot_dim - 1.0);
        m = 0.1 * log(d->factor) + 1.0;
    }
    if (d->mscale != 0.0) m = d->mscale;
    if (rmoe_status s = check_device(d->device)) return s;
    std::vector<double> f;
    rmoe_rope* r = nullptr;
    try {
        f.resize(pairs);
        r = new rmoe_rope();
        r->own.ptrs.reserve(4);  // nothing below throws
    } catch (...) {
        delete r;
        return fail(RMOE_ERR_OOM, "rope handle");
    }
    for (uint32_t i = 0; i < pairs; i++) {
        double v = pow(d->base, -2.0 * i / d->rot_dim);
        if (d->scaling == RMOE_ROPE_LINEAR) v /= d->factor;
        if (d->scaling == RMOE_ROPE_YARN) {
            const double g = 1.0 - fmin(fmax((i - low) / fmax(high - low, 0.001), 0.0), 1.0);
            v = v * g + v / d->factor * (1.0 - g);
        }
        f[i] = d->freq_factors ? v / d->freq_factors[i] : v;
    }
    DeviceGuard g(d->device);
    r->device = d->device;
    r->rot = d->rot_dim;
    r->layout = d->layout;
    r->max_pos = d->max_pos;
    const uint64_t n = (uint64_t)d->max_pos * pairs;
    r->table = (float2*)r->own.alloc(n * sizeof(float2));
    double* fd = (double*)r->own.alloc(pairs * sizeof(double));
    r->status = (unsigned*)r->own.alloc(16);
    if (!r->table || !fd || !r->status) {
        delete r;
        cudaGetLastError();
        return fail(RMOE_ERR_OOM, "rope table: cudaMalloc(%llu) failed", (unsigned long long)(n * sizeof(float2)));
    }
    cudaError_t e = cudaMemcpy(fd, f.data(), pairs * sizeof(double), cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaMemset(r->status, 0, 16);
    if (e == cudaSuccess) {
        rope_table_kernel<<<(unsigned)((n + 255) / 256 < 148 * 16 ? (n + 255) / 256 : 148 * 16), 256>>>(r->table, fd,
                                                                                                   (int)pairs, n, m);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e != cudaSuccess) {
        delete r;
        return cuda_fail(e, "rope table");
    }
    *out = r;
    return RMOE_OK;
}

void rmoe_rope_destroy(rmoe_rope* r) {
    if (!r) return;
    DeviceGuard g(r->device);
    cudaDeviceSynchronize();
    delete r;
}

rmoe_status rmoe_rope_apply(rmoe_rope* r, const rmoe_rope_args* a, void* stream) {
    if (!r || !a) return fail(RMOE_ERR_INVALID, "null rope / arguments");
    if (!elt_ok(a->type)) return fail(RMOE_ERR_UNSUPPORTED, "rope: ggml type %u (F32, F16 or BF16)", a->type);
    if (a->head_dim < r->rot) return fail(RMOE_ERR_INVALID, "head_dim %u is below rot_dim %u", a->head_dim, r->rot);
    if (a->T > 0x7fffffffu || a->head_dim > 65536) return fail(RMOE_ERR_UNSUPPORTED, "rope: T %u x %u", a->T, a->head_dim);
    Rows q, qo, k, ko;
    rmoe_status s;
    if ((s = check_rows(a->q, a->T, a->type, "q", q)) || (s = check_rows(a->q_out, a->T, a->type, "q_out", qo)) ||
        (s = check_rows(a->k, a->T, a->type, "k", k)) || (s = check_rows(a->k_out, a->T, a->type, "k_out", ko)))
        return s;
    if (q.heads != qo.heads || k.heads != ko.heads) return fail(RMOE_ERR_INVALID, "rope: heads of the outputs differ");
    if (a->T == 0 || q.heads + k.heads == 0) return RMOE_OK;
    if (!a->positions) return fail(RMOE_ERR_INVALID, "null positions");
    DeviceGuard g(r->device);
    RopeArg ra{r->table, a->positions, (int)r->rot, r->layout == RMOE_ROPE_HALF, (int)r->max_pos,
               a->inverse ? -1.0f : 1.0f};
    cudaError_t e = launch_rope_apply(q, qo, k, ko, ra, (int)a->T, (int)a->head_dim, a->type, r->status,
                                      static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? RMOE_OK : cuda_fail(e, "rope launch");
}

rmoe_status rmoe_rope_status(rmoe_rope* r) {
    if (!r) return fail(RMOE_ERR_INVALID, "null rope");
    DeviceGuard g(r->device);
    unsigned hs = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpy(&hs, r->status, 4, cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && hs) e = cudaMemset(r->status, 0, 4);
    if (e == cudaSuccess && hs) e = cudaStreamSynchronize(cudaStreamLegacy);  // or it could clear a later call's error
    if (e != cudaSuccess) return cuda_fail(e, "rope status");
    if (hs) return fail(RMOE_ERR_DEVICE, "rope: device status 0x%x (a position outside the table)", hs);
    return RMOE_OK;
}

}  // extern "C"
