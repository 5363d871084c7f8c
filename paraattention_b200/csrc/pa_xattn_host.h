// Host side shared by the forward and the backward entry point of cross attention.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>

#include "../../include/pa_b200.h"
#include "pa_host.h"
#include "xattn_sm100.cuh"

namespace pa_host {

inline bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

inline int xattn_tensor(const void* p, const int64_t* stride, const char* what) {
    if (p == nullptr) return fail(PA_EINVAL, "xattn: %s is NULL", what);
    if (off16(p)) return fail(PA_EINVAL, "xattn: %s: base pointer must be 16-byte aligned", what);
    for (int i = 0; i < 3; ++i)
        if (stride[i] % 8 != 0) return fail(PA_EINVAL, "xattn: %s: byte stride %d must be a multiple of 16", what, i);
    return PA_OK;
}

inline int xattn_sizes(const pa_xattn_args* a) {
    if (a == nullptr) return fail(PA_EINVAL, "xattn: args is NULL");
    if (a->batch <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->seq_q <= 0 || a->seq_kv <= 0)
        return fail(PA_EINVAL, "xattn: batch, heads, kv_heads, seq_q and seq_kv must be positive");
    if (a->kv_batch != a->batch && a->kv_batch != 1) return fail(PA_EINVAL, "xattn: kv_batch must be batch or 1");
    if (a->heads % a->kv_heads != 0) return fail(PA_EINVAL, "xattn: heads must be a multiple of kv_heads");
    if (a->head_dim != 64 && a->head_dim != 128)
        return fail(PA_ENOTSUP, "xattn: head_dim %d: only 64 and 128 are built", a->head_dim);
    if (a->dtype != PA_BF16 && a->dtype != PA_F16) return fail(PA_EINVAL, "xattn: dtype must be PA_BF16 or PA_F16");
    if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return fail(PA_EINVAL, "xattn: scale must be positive and finite");
    // tile, row and step counts are 32-bit on the device; row and tile indexes run up to a tile past the end
    const double mt = std::ceil(a->seq_q / 128.0), kt = std::ceil(a->seq_kv / 128.0);
    if (double(a->batch) * a->heads * mt * 128 > 2147000000.0 || double(a->batch) * a->kv_heads * kt * 128 > 2147000000.0)
        return fail(PA_EINVAL, "xattn: problem too large for one launch");
    return PA_OK;
}

// Whole units or equal ranges of steps (see XSched)? Whole units take ceil(units / CTAs) rounds of
// `steps` steps; ranges take units * steps / CTAs steps plus what the partial results cost,
// `extra` steps' time and a thirty-second of the whole. `shared`: consecutive units that walk the same streamed tiles; they form teams
// unless that leaves more than one SM in sixteen without work.
inline pa::XSched xattn_schedule(long long units, long long steps, int shared, int sms, int extra, int* grid) {
    sms = std::min(sms, pa::kXMaxCtas);
    pa::XSched s;
    s.units = static_cast<int>(units);
    s.steps = static_cast<int>(steps);
    const long long all = units * steps;
    const long long whole = (units + sms - 1) / sms * steps, ranges = (all + sms - 1) / sms;
    s.split = whole - whole / 32 > ranges + extra ? 1 : 0;
    s.team = s.split && shared > 1 && shared <= sms && sms / shared * shared * 16 >= sms * 15 ? shared : 1;
    s.total = all / s.team;
    *grid = static_cast<int>(s.split ? std::min<long long>(sms / s.team, s.total) * s.team : std::min<long long>(sms, units));
    return s;
}

struct XattnMask {
    int64_t words_bytes = 0, bytes = 0;  // packed words, then one extent per batch entry
};
inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
inline XattnMask xattn_mask_layout(const pa_xattn_args* a) {
    XattnMask m;
    if (a->key_mask == nullptr) return m;
    m.words_bytes = up256(int64_t(a->batch) * ((a->seq_kv + 63) / 64) * 8);
    m.bytes = m.words_bytes + up256(int64_t(a->batch) * 4);
    return m;
}

// Sets a kernel's shared-memory limit, and whether its clusters may have more than 8 CTAs, once per device.
template <typename K>
int allow_smem(K kern, int bytes, const char* what, bool wide_clusters = false) {
    static std::mutex mu;
    static const void* done[64][32] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    const void* id = reinterpret_cast<const void*>(kern);
    std::lock_guard<std::mutex> g(mu);
    if (dev >= 0 && dev < 64)
        for (const void*& d : done[dev]) {
            if (d == id) return PA_OK;
            if (d == nullptr) break;
        }
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && wide_clusters) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return fail(PA_ECUDA, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64)
        for (const void*& d : done[dev])
            if (d == nullptr) {
                d = id;
                break;
            }
    return PA_OK;
}

inline int launched(const char* what) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(PA_ECUDA, "%s launch: %s", what, cudaGetErrorString(e));
    return PA_OK;
}

}  // namespace pa_host
