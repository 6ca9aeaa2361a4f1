// kv_attend.cu -- attention over the 8-bit paged cache: checks, and the choice of kernel.
#include <algorithm>
#include <cmath>

#include "kv_attend.h"

using namespace rmoe;

// The workspace for a call on stream s.
static rmoe_status split_ws(rmoe_kv* kv, cudaStream_t s, SplitWs& ws) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    cudaError_t e = cudaStreamIsCapturing(s, &cap);
    const SplitSlot::Use use = cap == cudaStreamCaptureStatusNone ? SplitSlot::CALLS : SplitSlot::GRAPHS;
    // while it captures, a stream may not be asked for its id
    if (use == SplitSlot::GRAPHS) id = reinterpret_cast<uintptr_t>(s);
    else if (e == cudaSuccess) e = cudaStreamGetId(s, &id);
    if (e != cudaSuccess) return cuda_fail(e, "kv attend stream");
    const std::lock_guard<std::mutex> lock(kv->slots_mu);
    SplitSlot* free_slot = nullptr;
    auto look = [&]() -> SplitSlot* {
        for (int i = 0; i < kv->n_slots; i++) {
            if (kv->slots[i].use == use && kv->slots[i].stream == id) return &kv->slots[i];
            if (kv->slots[i].use == SplitSlot::FREE) free_slot = &kv->slots[i];
        }
        return nullptr;
    };
    SplitSlot* slot = look();
    if (!slot && !free_slot && kv->n_slots < MAX_SPLIT_SLOTS) {
        if ((e = add_split_slot(kv)) != cudaSuccess) {
            cudaGetLastError();
            return fail(RMOE_ERR_OOM, "kv attend: workspace for another stream: %s", cudaGetErrorString(e));
        }
        look();
    }
    if (!slot && !free_slot && use == SplitSlot::CALLS) {
        // every slot is taken: once the device is done, those of plain calls are free again
        if ((e = cudaDeviceSynchronize()) != cudaSuccess) return cuda_fail(e, "kv attend");
        for (int i = 0; i < kv->n_slots; i++)
            if (kv->slots[i].use == SplitSlot::CALLS) kv->slots[i].use = SplitSlot::FREE;
        look();
    }
    if (!slot) {
        if (!free_slot)
            return fail(RMOE_ERR_UNSUPPORTED, "kv attend: calls on one cache from more than %d streams", MAX_SPLIT_SLOTS);
        slot = free_slot;
        slot->use = use;
        slot->stream = id;
    }
    ws = slot->ws;
    return RMOE_OK;
}

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
    if (!std::isfinite(a->scale)) return fail(RMOE_ERR_INVALID, "attention scale %g", a->scale);
    if ((uint64_t)a->T * (a->q.heads / kv->heads) > 0x7fffffffull)  // rows are numbered in 32 bits
        return fail(RMOE_ERR_UNSUPPORTED, "%u tokens x %u query heads per kv head", a->T, a->q.heads / kv->heads);
    if (a->T == 0) return RMOE_OK;
    if (a->R == 0) return fail(RMOE_ERR_INVALID, "tokens without requests");
    if (!a->lens || !a->cu || (a->max_blocks && !a->table)) return fail(RMOE_ERR_INVALID, "kv attend: null pointer");
    p.table = a->table; p.lens = a->lens; p.cu = a->cu; p.lse = a->lse;
    p.R = (int)a->R; p.max_blocks = (int)a->max_blocks; p.T = (int)a->T; p.scale = a->scale; p.window = (int)a->window;
    DeviceGuard g(kv->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const KvArg ka = kv_arg(kv);
    const uint64_t group = a->q.heads / kv->heads;
    p.group = (int)group;
    p.group_inv = group > 1 ? (uint32_t)((0xffffffffull + group) / group) : 0;
    if (group > 32768) return fail(RMOE_ERR_UNSUPPORTED, "%llu query heads per kv head", (unsigned long long)group);
    // Without a bound on any request's new tokens: one each when there are as many tokens as
    // requests.  A wrong guess costs time only, the split kernel takes whatever the other does not.
    const uint64_t longest = std::min<uint64_t>(a->max_new ? a->max_new : a->T > a->R ? a->T : 1, a->T);
    p.prompts = kv->dim <= 128 && longest * group >= PROMPT_MIN_ROWS &&
                (a->T * group / PROMPT_PAIR_ROWS + std::min(a->R, a->T)) * kv->heads >= PROMPT_MIN_CTAS;
    SplitWs ws{};
    if ((st = split_ws(kv, s, ws))) return st;
    cudaError_t e = p.prompts ? launch_prompt(kv->prompt_maps, ka, p, a->type, (int)kv->code, s) : cudaSuccess;
    // 16 rows per item where a request has more than 8 on average: the cache is read once for them.  8 / 16
    // rows per item in us (B200, 8 requests of 8192 tokens, 4 kv heads): bf16 of 128, 16 rows 34.7 / 37.0, 32
    // rows 56.1 / 48.1; of 64, 28.1 / 29.9 and 43.3 / 37.0; f32 of 64, 30.7 / 29.8 and 48.5 / 42.4; f32 of 128,
    // whose 16-row kernel spills 340 to 380 bytes a thread, 40.0 / 47.9 and 65.4 / 68.6.
    const uint64_t mean = group * (p.prompts ? 1 : (a->T + a->R - 1) / a->R);
    const int nr = mean > 8 && kv->dim <= 128 ? 16 : 8;
    if (e == cudaSuccess)
        e = launch_split(kv->split_maps, ka, p, ws, kv->sms, nr, a->type, (int)kv->code, s);
    return e == cudaSuccess ? RMOE_OK : cuda_fail(e, "kv attend launch");
}
