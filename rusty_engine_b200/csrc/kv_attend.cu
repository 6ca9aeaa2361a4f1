// kv_attend.cu -- attention over the 8-bit paged cache: checks, and the choice of kernel.
#include "kv_attend.h"

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
    p.split_rows = INT64_MAX;
    // 16 rows per item where a request has more than 8 on average: the cache is read once for them
    const uint64_t group = a->q.heads / kv->heads, mean = group * ((a->T + a->R - 1) / a->R);
    const int nr = mean > 8 && kv->dim <= 128 ? 16 : 8;
    cudaError_t e = launch_split(kv->split_maps, ka, p, SplitWs{kv->split_part, kv->split_ticket}, kv->sms, nr, a->type,
                                 (int)kv->code, s);
    return e == cudaSuccess ? RMOE_OK : cuda_fail(e, "kv attend launch");
}
