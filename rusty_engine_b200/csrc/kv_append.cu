// kv_append.cu -- writing new keys and values into the 8-bit paged cache, and reading them back.
#include "kv_code.cuh"
#include "rope.cuh"

namespace rmoe {

struct AppendArg {
    Rows k, v;
    const int32_t* slots;
    RopeArg rope;
    int T;
};

// One CTA per (token, head, K or V); the CTA of a run's first token writes the whole run, the
// others return.  Two passes over the run's elements: the largest magnitude, then the codes.
template <typename T, int CODE>
__global__ void __launch_bounds__(128) kv_append_kernel(KvArg kv, AppendArg a) {
    const int t0 = blockIdx.x, h = blockIdx.y, isv = blockIdx.z, tid = threadIdx.x;
    const int bs = kv.bs, dim = kv.dim;
    pdl_trigger();
    pdl_wait();
    const int slot = __ldg(a.slots + t0);
    if (slot < 0) return;
    const int first = slot & (bs - 1), block = slot / bs;
    if (block >= kv.n_blocks) {
        if (tid == 0 && h == 0) atomicOr(kv.status, (unsigned)DERR_INDEX);
        return;
    }
    if (first != 0 && t0 > 0 && __ldg(a.slots + t0 - 1) == slot - 1) return;  // inside a run
    int n = 1;
    while (first + n < bs && t0 + n < a.T && __ldg(a.slots + t0 + n) == slot + n) n++;

    const Rows& in = isv ? a.v : a.k;
    const int units = dim / 16;
    const bool rot = !isv && a.rope.table;
    auto load = [&](int i, float* v, int& ca, int& cb) {  // unit i of the run
        const int j = i / units, u = i - j * units, t = t0 + j;
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
    float amax = 0.0f;
    bool bad = false;
    for (int i = tid; i < n * units; i += 128) {
        float v[16];
        int ca, cb;
        load(i, v, ca, cb);
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float m = fabsf(v[e]);
            if (m <= 3.4028234663852886e38f) amax = fmaxf(amax, m); else bad = true;
        }
    }
    __shared__ float red[4];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (bad) atomicOr(kv.status, (unsigned)DERR_NONFINITE);
    if ((tid & 31) == 0) red[tid >> 5] = amax;
    float* sp = (isv ? kv.vs : kv.ks) + (size_t)block * kv.heads + h;
    const float old = first ? *sp : 0.0f;
    __syncthreads();
    amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float want = __fmul_rn(amax, Code<CODE>::PER);
    if (want < 1.1754943508222875e-38f) want = 0.0f;  // 1 / want must stay finite
    const float scale = fmaxf(old, want), inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    uint8_t* base = (isv ? kv.v : kv.k) + ((size_t)block * kv.heads + h) * bs * dim;
    if (scale > old && first) {  // the block's earlier tokens, rounded again to the new scale
        const float ratio = __fmul_rn(old, inv);
        for (int i = tid; i < first * dim / 4; i += 128) {
            uint32_t w = reinterpret_cast<uint32_t*>(base)[i], o = 0;
#pragma unroll
            for (int e = 0; e < 4; e++)
                o |= Code<CODE>::put(__fmul_rn(Code<CODE>::get(w >> (8 * e)), ratio)) << (8 * e);
            reinterpret_cast<uint32_t*>(base)[i] = o;
        }
    }
    for (int i = tid; i < n * units; i += 128) {
        float v[16];
        int ca, cb;
        const int j = load(i, v, ca, cb);
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; e++) w[e / 4] |= Code<CODE>::put(__fmul_rn(v[e], inv)) << (8 * (e & 3));
        uint8_t* row = base + (size_t)(first + j) * dim;
        *reinterpret_cast<uint2*>(row + ca) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(row + cb) = make_uint2(w[2], w[3]);
    }
    if (tid == 0) *sp = scale;  // every thread read the old one before the barrier
}

// One thread per 16 elements of a slot and head, K then V.
template <typename T, int CODE>
__global__ void __launch_bounds__(256) kv_read_kernel(KvArg kv, const int32_t* slots, int n, T* ko, T* vo) {
    pdl_trigger();
    pdl_wait();
    const int units = kv.dim / 16;
    const uint64_t per = (uint64_t)n * kv.heads * units, all = 2 * per;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < all; i += gridDim.x * 256ull) {
        const bool isv = i >= per;
        const uint64_t r = isv ? i - per : i;
        const int u = (int)(r % units);
        const uint64_t th = r / units;
        const int h = (int)(th % kv.heads), t = (int)(th / kv.heads);
        const int slot = __ldg(slots + t);
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] = 0.0f;
        if (slot >= 0 && slot / kv.bs < kv.n_blocks) {
            const size_t bh = (size_t)(slot / kv.bs) * kv.heads + h;
            const float s = __ldg((isv ? kv.vs : kv.ks) + bh);
            const uint4 w = __ldg(reinterpret_cast<const uint4*>((isv ? kv.v : kv.k) + (bh * kv.bs + (slot & (kv.bs - 1))) * kv.dim) + u);
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 16; e++) v[e] = __fmul_rn(Code<CODE>::get(ww[e / 4] >> (8 * (e & 3))), s);
        } else if (slot >= 0 && u == 0 && h == 0) {
            atomicOr(kv.status, (unsigned)DERR_INDEX);
        }
        T* y = (isv ? vo : ko) + th * kv.dim + 16 * u;
        store8(y, true, v);
        store8(y + 8, true, v + 8);
    }
}

template <typename T, int CODE>
static cudaError_t append_launch(const KvArg& kv, const AppendArg& a, cudaStream_t s) {
    return launch_pdl(kv_append_kernel<T, CODE>, dim3((unsigned)a.T, (unsigned)kv.heads, 2), dim3(128), 0, s, kv, a);
}

template <typename T, int CODE>
static cudaError_t read_launch(const KvArg& kv, const int32_t* slots, int n, void* ko, void* vo, cudaStream_t s) {
    const uint64_t all = 2ull * n * kv.heads * (kv.dim / 16), ctas = (all + 255) / 256;
    return launch_pdl(kv_read_kernel<T, CODE>, dim3((unsigned)(ctas < 148 * 64 ? ctas : 148 * 64)), dim3(256), 0, s, kv, slots, n,
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
    Rows q, qo;
    rmoe_status st;
    if ((st = check_rows(a->k, a->T, a->type, "k", p.k)) || (st = check_rows(a->v, a->T, a->type, "v", p.v)) ||
        (st = check_rows(a->q, a->T, a->type, "q", q)) || (st = check_rows(a->q_out, a->T, a->type, "q_out", qo)))
        return st;
    if (a->k.heads != kv->heads || a->v.heads != kv->heads)
        return fail(RMOE_ERR_INVALID, "k / v have %u / %u heads, the cache %u", a->k.heads, a->v.heads, kv->heads);
    if (q.heads != qo.heads) return fail(RMOE_ERR_INVALID, "q_out has %d heads, q %d", qo.heads, q.heads);
    if (q.heads && !a->rope) return fail(RMOE_ERR_INVALID, "q is only taken with a rope");
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
    cudaError_t e = cudaSuccess;
    if (q.heads) {
        Rows none{};
        e = launch_rope_apply(q, qo, none, none, p.rope, p.T, ka.dim, a->type, kv->status, s);
    }
    if (e == cudaSuccess) {
        if (a->type == T_F32)
            e = i8 ? append_launch<float, RMOE_KV_INT8>(ka, p, s) : append_launch<float, RMOE_KV_E4M3>(ka, p, s);
        else if (a->type == T_F16)
            e = i8 ? append_launch<__half, RMOE_KV_INT8>(ka, p, s) : append_launch<__half, RMOE_KV_E4M3>(ka, p, s);
        else
            e = i8 ? append_launch<__nv_bfloat16, RMOE_KV_INT8>(ka, p, s)
                   : append_launch<__nv_bfloat16, RMOE_KV_E4M3>(ka, p, s);
    }
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
