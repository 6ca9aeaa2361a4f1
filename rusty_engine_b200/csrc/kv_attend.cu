// kv_attend.cu -- attention over the 8-bit paged cache.
//
// out_i = sum_j softmax_j(scale ks_b(j) q_i . kc_j) vs_b(j) vc_j over the keys that query i sees.
// One CTA per (token, query head), four warps that take every fourth key, lanes over the head's
// elements; each warp keeps a running maximum, sum and output, joined at the end.
#include "kv_code.cuh"
#include "rope.cuh"

namespace rmoe {

struct AttendArg {
    Rows q, out;
    const int32_t *table, *lens, *cu;
    float* lse;
    int R, max_blocks, T;
    float scale;
    int window;
};

template <typename T, int CODE, int DIM>
__global__ void __launch_bounds__(128) kv_attend_simple_kernel(KvArg kv, AttendArg a) {
    constexpr int PER = DIM / 32;
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int group = a.q.heads / kv.heads, kh = h / group, bs = kv.bs;
    // the request of token t
    int lo = 0, hi = a.R - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(a.cu + mid) <= t) lo = mid; else hi = mid - 1;
    }
    const int r = lo;
    int j0 = 0, j1 = 0;  // the keys it sees
    if (t >= __ldg(a.cu + r) && t < __ldg(a.cu + r + 1)) {
        const int pos = __ldg(a.lens + r) - __ldg(a.cu + r + 1) + t;
        j1 = (int)min((int64_t)pos + 1, (int64_t)a.max_blocks * bs);
        j0 = a.window ? max(0, pos - a.window + 1) : 0;
    }
    float q[PER], o[PER], m = -INFINITY, l = 0.0f;
    const T* qp = reinterpret_cast<const T*>(a.q.p) + t * a.q.st + h * a.q.sh + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; i++) q[i] = Elt<T>::get(qp[i]), o[i] = 0.0f;
    for (int j = j0 + w; j < j1; j += 4) {
        const int b = __ldg(a.table + (size_t)r * a.max_blocks + j / bs);
        if ((unsigned)b >= (unsigned)kv.n_blocks) {
            if (lane == 0) atomicOr(kv.status, (unsigned)DERR_INDEX);
            continue;
        }
        const size_t bh = (size_t)b * kv.heads + kh;
        const uint8_t* kp = kv.k + (bh * bs + (j & (bs - 1))) * DIM + lane * PER;
        const uint8_t* vp = kv.v + (bh * bs + (j & (bs - 1))) * DIM + lane * PER;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) s = fmaf(q[i], Code<CODE>::get(kp[i]), s);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= __ldg(kv.ks + bh) * a.scale;
        const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.0f : expf(m - mn), p = expf(s - mn), pv = p * __ldg(kv.vs + bh);
        m = mn;
        l = l * c + p;
#pragma unroll
        for (int i = 0; i < PER; i++) o[i] = fmaf(pv, Code<CODE>::get(vp[i]), o[i] * c);
    }
    __shared__ float sm[4], sl[4], so[4][DIM];
    if (lane == 0) sm[w] = m, sl[w] = l;
#pragma unroll
    for (int i = 0; i < PER; i++) so[w][lane * PER + i] = o[i];
    __syncthreads();
    const float mm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float c[4], ll = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        c[i] = sm[i] == -INFINITY ? 0.0f : expf(sm[i] - mm);
        ll += sl[i] * c[i];
    }
    T* op = reinterpret_cast<T*>(a.out.p) + t * a.out.st + h * a.out.sh;
    for (int i = threadIdx.x; i < DIM; i += 128) {
        const float v = so[0][i] * c[0] + so[1][i] * c[1] + so[2][i] * c[2] + so[3][i] * c[3];
        op[i] = Elt<T>::put(ll > 0.0f ? v / ll : 0.0f);
    }
    if (threadIdx.x == 0 && a.lse) a.lse[(size_t)t * a.q.heads + h] = ll > 0.0f ? mm + logf(ll) : -INFINITY;
}

template <typename T, int CODE>
static cudaError_t attend_launch(const KvArg& kv, const AttendArg& a, cudaStream_t s) {
    const dim3 grid((unsigned)a.T, (unsigned)a.q.heads);
    if (kv.dim == 64)
        kv_attend_simple_kernel<T, CODE, 64><<<grid, 128, 0, s>>>(kv, a);
    else if (kv.dim == 128)
        kv_attend_simple_kernel<T, CODE, 128><<<grid, 128, 0, s>>>(kv, a);
    else
        kv_attend_simple_kernel<T, CODE, 256><<<grid, 128, 0, s>>>(kv, a);
    return cudaGetLastError();
}

}  // namespace rmoe

using namespace rmoe;

extern "C" rmoe_status rmoe_kv_attend(rmoe_kv* kv, const rmoe_kv_attend_args* a, void* stream) {
    if (!kv || !a) return fail(RMOE_ERR_INVALID, "null cache / arguments");
    if (!elt_ok(a->type)) return fail(RMOE_ERR_UNSUPPORTED, "kv attend: ggml type %u (F32, F16 or BF16)", a->type);
    if (a->T > 0x7fffffffu || a->R > 0x7ffffffu || a->window > 0x7fffffffu || (uint64_t)a->max_blocks * kv->bs > 0x7fffffffull)
        return fail(RMOE_ERR_UNSUPPORTED, "kv attend: T %u, R %u, window %u, %u blocks in a row", a->T, a->R, a->window,
                    a->max_blocks);
    AttendArg p{};
    rmoe_status st;
    if ((st = check_rows(a->q, a->T, a->type, "q", p.q)) || (st = check_rows(a->out, a->T, a->type, "out", p.out))) return st;
    if (a->q.heads == 0 || a->q.heads % kv->heads)
        return fail(RMOE_ERR_INVALID, "%u query heads over %u kv heads", a->q.heads, kv->heads);
    if (a->out.heads != a->q.heads) return fail(RMOE_ERR_INVALID, "out has %u heads, q %u", a->out.heads, a->q.heads);
    if (a->T == 0) return RMOE_OK;
    if (a->R == 0) return fail(RMOE_ERR_INVALID, "tokens without requests");
    if (!a->lens || !a->cu || (a->max_blocks && !a->table)) return fail(RMOE_ERR_INVALID, "kv attend: null pointer");
    p.table = a->table; p.lens = a->lens; p.cu = a->cu; p.lse = a->lse;
    p.R = (int)a->R; p.max_blocks = (int)a->max_blocks; p.T = (int)a->T; p.scale = a->scale; p.window = (int)a->window;
    DeviceGuard g(kv->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const KvArg ka = kv_arg(kv);
    const bool i8 = kv->code == RMOE_KV_INT8;
    cudaError_t e;
    if (a->type == T_F32)
        e = i8 ? attend_launch<float, RMOE_KV_INT8>(ka, p, s) : attend_launch<float, RMOE_KV_E4M3>(ka, p, s);
    else if (a->type == T_F16)
        e = i8 ? attend_launch<__half, RMOE_KV_INT8>(ka, p, s) : attend_launch<__half, RMOE_KV_E4M3>(ka, p, s);
    else
        e = i8 ? attend_launch<__nv_bfloat16, RMOE_KV_INT8>(ka, p, s)
               : attend_launch<__nv_bfloat16, RMOE_KV_E4M3>(ka, p, s);
    return e == cudaSuccess ? RMOE_OK : cuda_fail(e, "kv attend launch");
}
