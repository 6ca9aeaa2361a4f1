// kv.cu -- the paged 8-bit KV cache handle: memory, checks, status.
#include <algorithm>

#include "kv_attend.h"

namespace rmoe {

cudaError_t add_split_slot(rmoe_kv* kv) {
    const size_t bytes = kv->sms * split_part_bytes((int)kv->dim);
    // allowed while this or another thread captures a graph: nothing here belongs into one
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) return e;
    char* p = nullptr;
    cudaStream_t s = nullptr;
    e = cudaMalloc(&p, bytes + kv->sms * 4);
    // on a stream of its own, so that nothing queued elsewhere is waited for
    if (e == cudaSuccess) e = cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking);
    if (e == cudaSuccess) e = cudaMemsetAsync(p + bytes, 0, kv->sms * 4, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (s) cudaStreamDestroy(s);
    if (e == cudaSuccess)
        kv->slots[kv->n_slots++] = SplitSlot{SplitSlot::FREE, 0, SplitWs{(float*)p, (unsigned*)(p + bytes)}};
    else
        cudaFree(p);
    cudaThreadExchangeStreamCaptureMode(&mode);
    return e;
}

}  // namespace rmoe

using namespace rmoe;

extern "C" {

rmoe_status rmoe_kv_create(const rmoe_kv_desc* d, rmoe_kv** out) {
    if (!out) return fail(RMOE_ERR_INVALID, "null output handle");
    *out = nullptr;
    if (!d) return fail(RMOE_ERR_INVALID, "null cache description");
    if (!block_size_ok(d->block_size)) return fail(RMOE_ERR_UNSUPPORTED, "block size %u (16, 32, 64 or 128)", d->block_size);
    if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
        return fail(RMOE_ERR_UNSUPPORTED, "head_dim %u (64, 128 or 256)", d->head_dim);
    if (d->code > RMOE_KV_E4M3) return fail(RMOE_ERR_UNSUPPORTED, "cache code %u", d->code);
    if (d->n_blocks == 0 || d->n_kv_heads == 0 || d->n_kv_heads > 4096)
        return fail(RMOE_ERR_INVALID, "%u blocks, %u kv heads", d->n_blocks, d->n_kv_heads);
    const uint64_t rows = (uint64_t)d->n_blocks * d->n_kv_heads * d->block_size;
    if (rows > 0x7fffffffull)  // the row coordinate of a tile copy and a slot are 32-bit
        return fail(RMOE_ERR_UNSUPPORTED, "%u blocks x %u heads x %u tokens exceed 2^31 rows", d->n_blocks, d->n_kv_heads,
                    d->block_size);
    const int given = (d->k != nullptr) + (d->v != nullptr) + (d->k_scale != nullptr) + (d->v_scale != nullptr);
    if (given != 0 && given != 4) return fail(RMOE_ERR_INVALID, "give all of k, v, k_scale, v_scale or none");
    if ((reinterpret_cast<uintptr_t>(d->k) | reinterpret_cast<uintptr_t>(d->v)) & 15)
        return fail(RMOE_ERR_INVALID, "cache codes must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(d->k_scale) | reinterpret_cast<uintptr_t>(d->v_scale)) & 3)
        return fail(RMOE_ERR_INVALID, "cache scales must be 4-byte aligned");
    if (rmoe_status s = check_device(d->device)) return s;
    DeviceGuard g(d->device);
    rmoe_kv* kv = nullptr;
    try {
        kv = new rmoe_kv();
        kv->own.ptrs.reserve(8);  // nothing below throws
    } catch (...) {
        delete kv;
        return fail(RMOE_ERR_OOM, "cache handle");
    }
    kv->device = d->device;
    kv->n_blocks = d->n_blocks;
    kv->bs = d->block_size;
    kv->heads = d->n_kv_heads;
    kv->dim = d->head_dim;
    kv->code = d->code;
    const uint64_t bytes = rows * d->head_dim, sb = (uint64_t)d->n_blocks * d->n_kv_heads * 4;
    cudaDeviceGetAttribute(&kv->sms, cudaDevAttrMultiProcessorCount, d->device);
    kv->status = (unsigned*)kv->own.alloc(16);
    bool ok = kv->status && add_split_slot(kv) == cudaSuccess;
    cudaError_t e = ok ? cudaMemset(kv->status, 0, 16) : cudaSuccess;
    if (given) {
        kv->k = (uint8_t*)d->k;
        kv->v = (uint8_t*)d->v;
        kv->ks = d->k_scale;
        kv->vs = d->v_scale;
    } else if (ok) {
        kv->k = (uint8_t*)kv->own.alloc(bytes);
        kv->v = (uint8_t*)kv->own.alloc(bytes);
        kv->ks = (float*)kv->own.alloc(sb);
        kv->vs = (float*)kv->own.alloc(sb);
        ok = kv->k && kv->v && kv->ks && kv->vs;
        if (ok && e == cudaSuccess) e = cudaMemset(kv->k, 0, bytes);
        if (ok && e == cudaSuccess) e = cudaMemset(kv->v, 0, bytes);
        if (ok && e == cudaSuccess) e = cudaMemset(kv->ks, 0, sb);
        if (ok && e == cudaSuccess) e = cudaMemset(kv->vs, 0, sb);
    }
    // a memset does not wait for the device, and non-blocking streams do not wait for its stream: the
    // first call on one of those must not overtake it
    if (ok && e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);
    if (!ok || e != cudaSuccess) {
        delete kv;
        cudaGetLastError();
        return ok ? cuda_fail(e, "cache memory")
                  : fail(RMOE_ERR_OOM, "cache memory: cudaMalloc of 2 x %llu bytes failed", (unsigned long long)bytes);
    }
    const uint32_t box = std::min<uint32_t>(kv->bs, split_tile_tokens((int)kv->dim));
    if (!make_code_map(kv->k, rows, kv->dim, box, kv->split_maps.k) || !make_code_map(kv->v, rows, kv->dim, box, kv->split_maps.v) ||
        !make_code_map(kv->k, rows, kv->dim, kv->bs, kv->prompt_maps.k) || !make_code_map(kv->v, rows, kv->dim, kv->bs, kv->prompt_maps.v)) {
        delete kv;
        return fail(RMOE_ERR_CUDA, "cuTensorMapEncodeTiled failed for the cache");
    }
    *out = kv;
    return RMOE_OK;
}

void rmoe_kv_destroy(rmoe_kv* kv) {
    if (!kv) return;
    DeviceGuard g(kv->device);
    cudaDeviceSynchronize();
    delete kv;
}

rmoe_status rmoe_kv_buffers(const rmoe_kv* kv, rmoe_kv_desc* d) {
    if (!kv || !d) return fail(RMOE_ERR_INVALID, "null cache / description");
    *d = rmoe_kv_desc{kv->n_blocks, kv->bs, kv->heads, kv->dim, kv->code, kv->device, kv->k, kv->v, kv->ks, kv->vs};
    return RMOE_OK;
}

rmoe_status rmoe_kv_status(rmoe_kv* kv) {
    if (!kv) return fail(RMOE_ERR_INVALID, "null cache");
    DeviceGuard g(kv->device);
    unsigned hs = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpy(&hs, kv->status, 4, cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && hs) e = cudaMemset(kv->status, 0, 4);
    if (hs & DERR_TIMEOUT) {
        // CTAs of a call whose waits ran out may not have been counted: the next call starts from 0 again
        const std::lock_guard<std::mutex> lock(kv->slots_mu);
        for (int i = 0; i < kv->n_slots && e == cudaSuccess; i++) e = cudaMemset(kv->slots[i].ws.ticket, 0, kv->sms * 4);
    }
    if (e == cudaSuccess && hs) e = cudaStreamSynchronize(cudaStreamLegacy);  // or it could clear a later call's error
    if (e != cudaSuccess) return cuda_fail(e, "cache status");
    if (hs)
        return fail(RMOE_ERR_DEVICE, "kv cache: device status 0x%x%s%s%s", hs,
                    (hs & DERR_INDEX) ? " (a slot, block or position out of range)" : "",
                    (hs & DERR_NONFINITE) ? " (a key or value that is not finite)" : "",
                    (hs & DERR_TIMEOUT) ? " (a bounded wait ran out)" : "");
    return RMOE_OK;
}

rmoe_status rmoe_selftest_kv_lost_wait(rmoe_kv* kv) {
    if (!kv) return fail(RMOE_ERR_INVALID, "null cache");
    DeviceGuard g(kv->device);
    const std::lock_guard<std::mutex> lock(kv->slots_mu);
    const unsigned hs = DERR_TIMEOUT;
    cudaError_t e = cudaDeviceSynchronize();
    for (int i = 0; i < kv->n_slots && e == cudaSuccess; i++) e = cudaMemset(kv->slots[i].ws.ticket, 1, kv->sms * 4);
    if (e == cudaSuccess) e = cudaMemcpy(kv->status, &hs, 4, cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    return e == cudaSuccess ? RMOE_OK : cuda_fail(e, "kv self-test");
}

}  // extern "C"
