// kv_append.cu -- writing new keys and values into the 8-bit paged cache, and reading them back.
#include <algorithm>

#include "kv_code.cuh"
#include "rope.cuh"

namespace rmoe {

struct AppendArg {
    Rows k, v, q, qo;
    const int32_t* slots;
    RopeArg rope;
    int T;
    int window;   // tokens of a CTA's window
    int kv_ctas;  // the CTAs from here on turn q
    bool apart;   // q is turned by the kernel before this one, which had its inputs when it let this one start
};

// A run is the tokens of one call that go to consecutive slots of one block: they share a scale.
// A CTA looks at `window` tokens for one head of K or V and writes the runs that begin there: all
// threads together where few begin (prompts), a warp per run where many do (decoded tokens).
// A run is bound by reading its elements once; up to HOLD units of 16 are held by a thread between the
// pass that finds the largest magnitude and the pass that rounds, the rest is read again (L2).  Three CTAs an
// SM leave a thread 80 registers, and 84 (f32) or 96 bytes of it spill.
// Measured (B200): 8192 tokens of 4 + 4 heads of 128 in bf16 with rope, blocks of 64: 15.7 us, 25 MB, 1.6
// TB/s (12.7 us without rope); it waits for its loads (slots, then elements and positions, then angles:
// three trips, 21 warps an SM).  32 decoded tokens of f32 with the read of them: 5.8 us, latency.
static constexpr int APT = 256, HOLD = 2;

// Writes the run of n tokens from t0 on, at slot; thread i of NT.  red: a word per warp (NT > 32).
template <typename T, int CODE, int NT>
__device__ __forceinline__ void write_run(const KvArg& kv, const AppendArg& a, bool isv, int h, int t0, int n, int slot, int tid,
                                          float* red) {
    const int bs = kv.bs, dim = kv.dim, units = dim >> 4, lu = 31 - __clz(units);  // dim is a power of two
    const int first = slot & (bs - 1), block = slot >> kv.shift;
    const Rows& in = isv ? a.v : a.k;
    const bool rot = !isv && a.rope.table;
    auto load = [&](int i, float* v, int& ca, int& cb) {  // unit i of the run
        const int j = i >> lu, u = i & (units - 1);
        const int64_t t = t0 + j;
        unit_chunks(u, rot ? a.rope.rot : 0, a.rope.half, ca, cb);
        const T* x = reinterpret_cast<const T*>(in.p) + t * in.st + h * in.sh;
        load8(x + ca, in.vec, v);
        load8(x + cb, in.vec, v + 8);
        if (rot) {
            const int p = __ldg(a.rope.pos + t);
            if ((unsigned)p < (unsigned)a.rope.max_pos)
                turn_unit(v, u, a.rope.table + (size_t)p * (a.rope.rot / 2), a.rope.rot, a.rope.half, 1.0f);
            else if (u == 0 && h == 0)
                atomicOr(kv.status, (unsigned)DERR_INDEX);
        }
        return j;
    };
    float* sp = (isv ? kv.vs : kv.ks) + (size_t)block * kv.heads + h;
    const float old = first ? *sp : 0.0f;
    float amax = 0.0f, held[HOLD][16];
    bool bad = false;
    auto top = [&](const float* v) {
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float m = fabsf(v[e]);
            if (m <= 3.4028234663852886e38f) amax = fmaxf(amax, m); else bad = true;
        }
    };
    int ca, cb;
#pragma unroll
    for (int k = 0; k < HOLD; k++)
        if (tid + k * NT < n * units) load(tid + k * NT, held[k], ca, cb);
#pragma unroll
    for (int k = 0; k < HOLD; k++)
        if (tid + k * NT < n * units) top(held[k]);
    for (int i = tid + HOLD * NT; i < n * units; i += NT) {
        float v[16];
        load(i, v, ca, cb);
        top(v);
    }
    if (bad) atomicOr(kv.status, (unsigned)DERR_NONFINITE);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (NT > 32) {
        if ((tid & 31) == 0) red[tid >> 5] = amax;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NT / 32; i++) amax = fmaxf(amax, red[i]);
    }
    float want = __fmul_rn(amax, Code<CODE>::PER);
    if (want < 1.1754943508222875e-38f) want = 0.0f;  // 1 / want must stay finite
    const float scale = fmaxf(old, want), inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    uint8_t* base = (isv ? kv.v : kv.k) + ((size_t)block * kv.heads + h) * bs * dim;
    if (scale > old && first) {  // the block's earlier tokens, rounded again to the new scale
        const float ratio = __fmul_rn(old, inv);
        for (int i = tid; i < first * dim / 4; i += NT) {
            const uint32_t w = reinterpret_cast<uint32_t*>(base)[i];
            uint32_t o = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) o |= Code<CODE>::put(__fmul_rn(Code<CODE>::get(w >> (8 * e)), ratio)) << (8 * e);
            reinterpret_cast<uint32_t*>(base)[i] = o;
        }
    }
    auto store = [&](int i, const float* v) {
        const int j = i >> lu, u = i & (units - 1);
        unit_chunks(u, rot ? a.rope.rot : 0, a.rope.half, ca, cb);
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; e++) w[e / 4] |= Code<CODE>::put(__fmul_rn(v[e], inv)) << (8 * (e & 3));
        uint8_t* row = base + (size_t)(first + j) * dim;
        *reinterpret_cast<uint2*>(row + ca) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(row + cb) = make_uint2(w[2], w[3]);
    };
#pragma unroll
    for (int k = 0; k < HOLD; k++)
        if (tid + k * NT < n * units) store(tid + k * NT, held[k]);
    for (int i = tid + HOLD * NT; i < n * units; i += NT) {
        float v[16];
        load(i, v, ca, cb);
        store(i, v);
    }
    if (NT > 32) __syncthreads();  // red is used again; every thread has read the old scale
    else __syncwarp();
    if (tid == 0) *sp = scale;
}

template <typename T, int CODE>
__global__ void __launch_bounds__(APT, 3) kv_append_kernel(KvArg kv, AppendArg a) {
    __shared__ float red[APT / 32];
    __shared__ int s_run[128], s_slot[128], s_n;  // the runs that begin in the window: first token and slot
    __shared__ unsigned s_cont[APT / 32];
    const int tid = threadIdx.x;
    pdl_trigger();
    if (!a.apart) pdl_wait();
    if ((int)blockIdx.x >= a.kv_ctas) {  // q, as the rope kernel turns it
        Rows none{};
        turn_items<T>(a.q, a.qo, none, none, a.rope, a.T, kv.dim, (int64_t)(blockIdx.x - a.kv_ctas) * APT + tid,
                      (int64_t)(gridDim.x - a.kv_ctas) * APT, kv.status);
        return;
    }
    const int per = 2 * kv.heads, win = blockIdx.x / per, hv = blockIdx.x - win * per, h = hv >> 1, bs = kv.bs;
    const bool isv = hv & 1;
    // the window's slots and those that a run beginning in it can reach (window + bs <= 256): which
    // of them continue their predecessor's run
    const int t = win * a.window + tid;
    const int slot = t < a.T ? __ldg(a.slots + t) : -1, prev = t > 0 && t < a.T ? __ldg(a.slots + t - 1) : -2;
    const bool cont = slot >= 0 && (slot & (bs - 1)) != 0 && prev == slot - 1;
    const unsigned cm = __ballot_sync(0xffffffffu, cont);
    if ((tid & 31) == 0) s_cont[tid >> 5] = cm;
    if (tid == 0) s_n = 0;
    __syncthreads();
    if (tid < a.window && slot >= 0 && !cont) {
        if ((slot >> kv.shift) < kv.n_blocks) {
            const int i = atomicAdd(&s_n, 1);
            s_run[i] = tid;
            s_slot[i] = slot;
        } else if (hv == 0) {
            atomicOr(kv.status, (unsigned)DERR_INDEX);
        }
    }
    __syncthreads();
    const int runs = s_n, lane = tid & 31, w = tid >> 5;
    // the run that begins at token x of the window: 1 + the bits that are set from x + 1 on
    auto length = [&](int x) {
        int n = 1;
        for (int b = x + 1;; b = (b | 31) + 1) {
            if (b >= APT) return n;
            const unsigned rest = ~(s_cont[b >> 5] >> (b & 31));  // first clear bit from b on
            const int ones = rest ? __ffs(rest) - 1 : 32, room = 32 - (b & 31);
            n += min(ones, room);
            if (ones < room) return n;
        }
    };
    if (runs <= 2) {
        for (int i = 0; i < runs; i++) {
            write_run<T, CODE, APT>(kv, a, isv, h, win * a.window + s_run[i], length(s_run[i]), s_slot[i], tid, red);
        }
    } else {
        for (int i = w; i < runs; i += APT / 32) {
            write_run<T, CODE, 32>(kv, a, isv, h, win * a.window + s_run[i], length(s_run[i]), s_slot[i], lane, nullptr);
        }
    }
    if (a.apart) pdl_wait();  // the next kernel may take the end of this one for the end of both
}

// One thread per 16 elements of a slot and head, K then V.  8192 slots of 4 heads of 128 as bf16: 6.8
// us, 25 MB, 3.7 TB/s; as f32 11.9 us, 42 MB (B200): a thread waits for its slot and then for its scale and
// codes, with nothing else of it in flight.
template <typename T, int CODE>
__global__ void __launch_bounds__(256) kv_read_kernel(KvArg kv, const int32_t* slots, int n, T* ko, T* vo) {
    pdl_trigger();
    pdl_wait();
    const int units = kv.dim / 16, lu = 31 - __clz(units);
    const bool isv = blockIdx.y;
    const uint64_t per = (uint64_t)n * kv.heads << lu;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < per; i += gridDim.x * 256ull) {
        const int u = (int)i & (units - 1);
        const uint64_t th = i >> lu;
        const int t = (th >> 32) == 0 ? (int)((uint32_t)th / (uint32_t)kv.heads) : (int)(th / kv.heads), h = (int)(th - (uint64_t)t * kv.heads);
        const int slot = __ldg(slots + t);
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] = 0.0f;
        if (slot >= 0 && (slot >> kv.shift) < kv.n_blocks) {
            const size_t bh = (size_t)(slot >> kv.shift) * kv.heads + h;
            const float s = __ldg((isv ? kv.vs : kv.ks) + bh);
            const uint4 w = __ldg(reinterpret_cast<const uint4*>((isv ? kv.v : kv.k) + (bh * kv.bs + (slot & (kv.bs - 1))) * kv.dim) + u);
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 16; e++) v[e] = __fmul_rn(Code<CODE>::get(ww[e / 4] >> (8 * (e & 3))), s);
        } else if (slot >= 0 && u == 0 && h == 0 && !isv) {
            atomicOr(kv.status, (unsigned)DERR_INDEX);
        }
        T* y = (isv ? vo : ko) + th * kv.dim + 16 * u;
        store8(y, true, v);
        store8(y + 8, true, v + 8);
    }
}

template <typename T, int CODE>
static cudaError_t append_launch(const KvArg& kv, AppendArg a, cudaStream_t s) {
    // Decoded tokens are a run each: windows of 8 give every warp one, until such windows fill the
    // chip; then a block's worth of tokens, in which a prompt begins one or two runs.  Windows of 8 / of a block
    // in us (B200, bf16, 4 heads of 128): 256 decoded tokens in blocks of 64 4.0 / 12.7, 1024 8.9 / 18.5, 4096
    // 28.9 / 28.5; in blocks of 16 1024 8.9 / 9.1, 4096 28.9 / 25.5.  Prompts in blocks of 64: 256 tokens 4.2 / 3.7,
    // 1024 6.3 / 5.0, 4096 13.8 / 7.5.  The rule goes by tokens alone, which only the device could tell
    // apart: from 1025 decoded tokens in blocks of 64 or 128 to some 4096 it loses up to 10 (128: 20) us.
    a.window = a.T <= 1024 ? 8 : kv.bs;
    const int64_t kvc = ((int64_t)a.T + a.window - 1) / a.window * kv.heads * 2;
    const int64_t qn = (int64_t)a.T * a.q.heads * (kv.dim / 16);
    // One launch for both where it is the launch that costs; for prompts q's stream goes through the
    // rope kernel's bulk copies, and this kernel runs beside it: neither needs the other's results.
    a.apart = qn > 148 * APT * 4;
    if (a.apart) {
        const Rows none{};
        cudaError_t e = launch_rope_apply(a.q, a.qo, none, none, a.rope, a.T, kv.dim, Elt<T>::TYPE, kv.status, s);
        if (e != cudaSuccess) return e;
    }
    const int64_t qc = a.apart ? 0 : (qn + APT - 1) / APT;
    if (kvc + qc > 0x7fffffff) return cudaErrorInvalidConfiguration;
    a.kv_ctas = (int)kvc;
    if (a.apart) {  // an SM runs both kernels at once only if they divide its memory alike
        static std::atomic<uint64_t> done{0};
        cudaError_t e = all_shared(kv_append_kernel<T, CODE>, done);
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(kv_append_kernel<T, CODE>, dim3((unsigned)(kvc + qc)), dim3(APT), 0, s, kv, a);
}

template <typename T, int CODE>
static cudaError_t read_launch(const KvArg& kv, const int32_t* slots, int n, void* ko, void* vo, cudaStream_t s) {
    const uint64_t ctas = ((uint64_t)n * kv.heads * (kv.dim / 16) + 255) / 256;
    return launch_pdl(kv_read_kernel<T, CODE>, dim3((unsigned)(ctas < 148 * 64 ? ctas : 148 * 64), 2), dim3(256), 0, s, kv, slots, n,
                      (T*)ko, (T*)vo);
}

}  // namespace rmoe

using namespace rmoe;

extern "C" {

rmoe_status rmoe_kv_append(rmoe_kv* kv, const rmoe_kv_append_args* a, void* stream) {
    if (!kv || !a) return fail(RMOE_ERR_INVALID, "null cache / arguments");
    if (!elt_ok(a->type)) return fail(RMOE_ERR_UNSUPPORTED, "kv append: ggml type %u (F32, F16 or BF16)", a->type);
    if (a->T > 0x7fffffffu) return fail(RMOE_ERR_UNSUPPORTED, "%u tokens", a->T);
    AppendArg p{};
    rmoe_status st;
    if ((st = check_rows(a->k, a->T, a->type, "k", p.k)) || (st = check_rows(a->v, a->T, a->type, "v", p.v)) ||
        (st = check_rows(a->q, a->T, a->type, "q", p.q)) || (st = check_rows(a->q_out, a->T, a->type, "q_out", p.qo)))
        return st;
    if (a->k.heads != kv->heads || a->v.heads != kv->heads)
        return fail(RMOE_ERR_INVALID, "k / v have %u / %u heads, the cache %u", a->k.heads, a->v.heads, kv->heads);
    if (p.q.heads != p.qo.heads) return fail(RMOE_ERR_INVALID, "q_out has %d heads, q %d", p.qo.heads, p.q.heads);
    if (p.q.heads && !a->rope) return fail(RMOE_ERR_INVALID, "q is only taken with a rope");
    if (a->rope) {
        if (a->rope->device != kv->device) return fail(RMOE_ERR_INVALID, "the rope is on another device");
        if (a->rope->rot > kv->dim || a->rope->rot % 16)
            return fail(RMOE_ERR_UNSUPPORTED, "rot_dim %u with head_dim %u (a multiple of 16, at most head_dim)", a->rope->rot,
                        kv->dim);
        if (a->T && !a->positions) return fail(RMOE_ERR_INVALID, "null positions");
    }
    if (a->T == 0) return RMOE_OK;
    if (!a->slots) return fail(RMOE_ERR_INVALID, "null slots");
    p.slots = a->slots;
    p.T = (int)a->T;
    if (a->rope) {
        p.rope = RopeArg{a->rope->table, a->positions, (int)a->rope->rot, a->rope->layout == RMOE_ROPE_HALF,
                         (int)a->rope->max_pos, 1.0f};
    }
    DeviceGuard g(kv->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const KvArg ka = kv_arg(kv);
    const bool i8 = kv->code == RMOE_KV_INT8;
    cudaError_t e;
    if (a->type == T_F32)
        e = i8 ? append_launch<float, RMOE_KV_INT8>(ka, p, s) : append_launch<float, RMOE_KV_E4M3>(ka, p, s);
    else if (a->type == T_F16)
        e = i8 ? append_launch<__half, RMOE_KV_INT8>(ka, p, s) : append_launch<__half, RMOE_KV_E4M3>(ka, p, s);
    else
        e = i8 ? append_launch<__nv_bfloat16, RMOE_KV_INT8>(ka, p, s) : append_launch<__nv_bfloat16, RMOE_KV_E4M3>(ka, p, s);
    return e == cudaSuccess ? RMOE_OK : cuda_fail(e, "kv append launch");
}

rmoe_status rmoe_kv_read(rmoe_kv* kv, const int32_t* slots, uint32_t n, uint32_t type, void* k_out, void* v_out,
                         void* stream) {
    if (!kv) return fail(RMOE_ERR_INVALID, "null cache");
    if (!elt_ok(type)) return fail(RMOE_ERR_UNSUPPORTED, "kv read: ggml type %u (F32, F16 or BF16)", type);
    if (n == 0) return RMOE_OK;
    if (n > 0x7fffffffu) return fail(RMOE_ERR_UNSUPPORTED, "%u slots", n);
    if (!slots || !k_out || !v_out) return fail(RMOE_ERR_INVALID, "kv read: null pointer");
    if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15)
        return fail(RMOE_ERR_INVALID, "kv read: outputs must be 16-byte aligned");
    DeviceGuard g(kv->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const KvArg ka = kv_arg(kv);
    const bool i8 = kv->code == RMOE_KV_INT8;
    const int m = (int)n;
    cudaError_t e;
    if (type == T_F32)
        e = i8 ? read_launch<float, RMOE_KV_INT8>(ka, slots, m, k_out, v_out, s)
               : read_launch<float, RMOE_KV_E4M3>(ka, slots, m, k_out, v_out, s);
    else if (type == T_F16)
        e = i8 ? read_launch<__half, RMOE_KV_INT8>(ka, slots, m, k_out, v_out, s)
               : read_launch<__half, RMOE_KV_E4M3>(ka, slots, m, k_out, v_out, s);
    else
        e = i8 ? read_launch<__nv_bfloat16, RMOE_KV_INT8>(ka, slots, m, k_out, v_out, s)
               : read_launch<__nv_bfloat16, RMOE_KV_E4M3>(ka, slots, m, k_out, v_out, s);
    return e == cudaSuccess ? RMOE_OK : cuda_fail(e, "kv read launch");
}

}  // extern "C"
