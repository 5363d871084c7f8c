// C ABI of cross attention, forward: argument validation, choice of the kernel, launches.
#include "pa_xattn_host.h"
#include "xattn_few_sm100.cuh"
#include "xattn_fwd_sm100.cuh"

using namespace pa_host;

namespace {

// Rows that share a key / value head: up to 16 take the kernel for few rows.
bool few_rows(const pa_xattn_args* a) {
    return static_cast<long long>(a->heads / a->kv_heads) * a->seq_q <= pa::kFewRows;
}

struct FwdPlan {
    pa::XSched sched;
    int grid = 0, mt = 0;
    int64_t off_ml = 0, off_o = 0, bytes = 0;
};

FwdPlan plan(const pa_xattn_args* a) {
    FwdPlan f;
    if (few_rows(a)) return f;
    f.mt = (a->seq_q + 127) / 128;
    const long long tiles = static_cast<long long>(a->heads / a->kv_heads) * f.mt;
    const long long units = (tiles + 1) / 2 * a->kv_heads * a->batch;
    f.sched = xattn_schedule(units, (a->seq_kv + 127) / 128, 1, sm_count(), 4, &f.grid);
    const int64_t mask = xattn_mask_layout(a).bytes;
    f.off_ml = mask;
    f.off_o = f.off_ml + (f.sched.split ? int64_t(f.grid) * 2 * 256 * 8 : 0);
    f.bytes = f.off_o + (f.sched.split ? int64_t(f.grid) * 2 * 256 * a->head_dim * 4 : 0);
    return f;
}

// CTAs per (batch, kv head) for `units` of them with `tiles` key tiles each: the least time by a model fitted to
// measurements (microseconds, head_dim 128; half the bytes at 64): 7 per CTA around its loop, 0.75 per tile,
// whole rounds of two CTAs per SM. Clusters of 16 take 12 more and compete for the few places with 16 free
// SMs: only where all of them run at once (8 units x 512 tiles 44 against 57 us with 8, but 32 units x 64
// tiles 42 against 19 us).
int few_cluster(long long units, int tiles, int head_dim, int sms) {
    const double scale = head_dim == 64 ? 0.5 : 1.0;
    double best = 0;
    int pick = 1;
    for (int c = 1; c <= pa::kFewMaxCluster && c <= tiles; c *= 2) {
        const long long ctas = units * c;
        if (c == 16 && ctas > sms) break;
        const double loop = scale * ((tiles + c - 1) / c);
        const double t = double((ctas + 2 * sms - 1) / (2 * sms)) * (loop * 0.75 + 7) + (c == 16 ? 12 : 0);
        if (c == 1 || t < best) {
            best = t;
            pick = c;
        }
    }
    return pick;
}

template <bool kBF16, int kD>
int run_few(const pa_xattn_args* a, cudaStream_t s) {
    pa::XFewParams p;
    memset(&p, 0, sizeof(p));
    p.q = static_cast<const uint16_t*>(a->q);
    p.k = static_cast<const uint16_t*>(a->k);
    p.v = static_cast<const uint16_t*>(a->v);
    p.out = static_cast<uint16_t*>(a->out);
    p.lse = a->lse;
    for (int i = 0; i < 3; ++i) {
        p.q_s[i] = a->q_stride[i];
        p.k_s[i] = (i == 0 && a->kv_batch == 1) ? 0 : a->k_stride[i];
        p.v_s[i] = (i == 0 && a->kv_batch == 1) ? 0 : a->v_stride[i];
        p.o_s[i] = a->o_stride[i];
    }
    p.mask = a->key_mask;
    p.mask_s = a->mask_stride;
    p.hkv = a->kv_heads;
    p.group = a->heads / a->kv_heads;
    p.sq = a->seq_q;
    p.skv = a->seq_kv;
    p.scale = a->scale;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.status = a->status;
    p.status_host = a->status_host;
    p.wait_ns = a->wait_limit_ns ? a->wait_limit_ns : 2000000000ull;
    const long long units = static_cast<long long>(a->batch) * a->kv_heads;
    const int tiles = (a->seq_kv + pa::kFewKeys - 1) / pa::kFewKeys;
    const int c = few_cluster(units, tiles, kD, sm_count());
    auto kern = pa::xattn_few_kernel<kBF16, kD>;
    const int smem = pa::few_smem_bytes<kD>();
    const int rc = allow_smem(kern, smem, "xattn few rows", true);
    if (rc != PA_OK) return rc;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(units * c));
    cfg.blockDim = dim3(2 * pa::kFewThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = c;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) return fail(PA_ECUDA, "xattn few rows launch: %s", cudaGetErrorString(e));
    return PA_OK;
}

template <bool kBF16, int kD>
int run_tiles(const pa_xattn_args* a, const FwdPlan& f, cudaStream_t s) {
    CUtensorMap mq, mk, mv, mo;
    int rc = make_map(&mq, a->q, a->dtype, kD, a->seq_q, a->heads, a->batch, 1, a->q_stride[2], a->q_stride[1], a->q_stride[0], 0, "q");
    if (rc == PA_OK) rc = make_map(&mk, a->k, a->dtype, kD, a->seq_kv, a->kv_heads, a->kv_batch, 1, a->k_stride[2], a->k_stride[1], a->k_stride[0], 0, "k");
    if (rc == PA_OK) rc = make_map(&mv, a->v, a->dtype, kD, a->seq_kv, a->kv_heads, a->kv_batch, 1, a->v_stride[2], a->v_stride[1], a->v_stride[0], 0, "v");
    if (rc == PA_OK) rc = make_map(&mo, a->out, a->dtype, kD, a->seq_q, a->heads, a->batch, 1, a->o_stride[2], a->o_stride[1], a->o_stride[0], 0, "out", 32, 32);
    if (rc != PA_OK) return rc;
    pa::XFwdParams p;
    memset(&p, 0, sizeof(p));
    p.kv_batch = a->kv_batch;
    p.hkv = a->kv_heads;
    p.group = a->heads / a->kv_heads;
    p.sq = a->seq_q;
    p.skv = a->seq_kv;
    p.mt = f.mt;
    p.scale = a->scale;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.out = static_cast<uint16_t*>(a->out);
    p.lse = a->lse;
    p.o_sb = a->o_stride[0];
    p.o_sh = a->o_stride[1];
    p.o_ss = a->o_stride[2];
    p.sched = f.sched;
    p.by_pairs = pa::x_div((p.group * f.mt + 1) / 2);
    p.by_hkv = pa::x_div(p.hkv);
    p.by_mt = pa::x_div(f.mt);
    p.status = a->status;
    p.status_host = a->status_host;
    p.wait_ns = a->wait_limit_ns ? a->wait_limit_ns : 2000000000ull;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    if (a->key_mask != nullptr) {
        p.words = reinterpret_cast<unsigned long long*>(ws);
        p.extent = reinterpret_cast<int*>(ws + xattn_mask_layout(a).words_bytes);
        pa::xattn_mask_kernel<<<a->batch, pa::kXMaskThreads, 0, s>>>(a->key_mask, a->mask_stride, a->seq_kv,
                                                                     reinterpret_cast<unsigned long long*>(ws),
                                                                     const_cast<int*>(p.extent));
        rc = launched("xattn mask");
        if (rc != PA_OK) return rc;
    }
    if (f.sched.split) {
        p.part_ml = reinterpret_cast<float2*>(ws + f.off_ml);
        p.part_o = reinterpret_cast<float*>(ws + f.off_o);
    }
    auto kern = pa::xattn_fwd_kernel<kBF16, kD>;
    rc = allow_smem(kern, pa::kXFwdSmemBytes, "xattn forward");
    if (rc != PA_OK) return rc;
    kern<<<f.grid, pa::kXFwdThreads, pa::kXFwdSmemBytes, s>>>(mq, mk, mv, mo, p);
    rc = launched("xattn forward");
    if (rc != PA_OK || !f.sched.split) return rc;
    pa::XCutList cuts;
    pa::x_list_cuts(f.sched, f.grid, &cuts);
    if (cuts.n == 0) return PA_OK;
    pa::xattn_fwd_join_kernel<kBF16, kD><<<dim3(cuts.n, kD / 8), 256, 0, s>>>(p, cuts);
    return launched("xattn forward join");
}

}  // namespace

extern "C" int64_t pa_xattn_bwd_workspace_bytes_(const pa_xattn_args* a);

extern "C" {

int64_t pa_xattn_workspace_bytes(const pa_xattn_args* a, int32_t backward) {
    const int rc = xattn_sizes(a);
    if (rc != PA_OK) return rc;
    return backward ? pa_xattn_bwd_workspace_bytes_(a) : plan(a).bytes;
}

int pa_xattn_fwd(const pa_xattn_args* a, void* stream) {
    int rc = xattn_sizes(a);
    if (rc == PA_OK) rc = xattn_tensor(a->q, a->q_stride, "q");
    if (rc == PA_OK) rc = xattn_tensor(a->k, a->k_stride, "k");
    if (rc == PA_OK) rc = xattn_tensor(a->v, a->v_stride, "v");
    if (rc == PA_OK) rc = xattn_tensor(a->out, a->o_stride, "out");
    if (rc != PA_OK) return rc;
    const FwdPlan f = plan(a);
    if (f.bytes > 0 && (a->workspace == nullptr || (reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0 || a->workspace_bytes < f.bytes))
        return fail(PA_EINVAL, "xattn: needs a 256-byte aligned workspace of %lld bytes", static_cast<long long>(f.bytes));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf16 = a->dtype == PA_BF16;
    if (few_rows(a)) {
        if (a->head_dim == 128) return bf16 ? run_few<true, 128>(a, s) : run_few<false, 128>(a, s);
        return bf16 ? run_few<true, 64>(a, s) : run_few<false, 64>(a, s);
    }
    if (a->head_dim == 128) return bf16 ? run_tiles<true, 128>(a, f, s) : run_tiles<false, 128>(a, f, s);
    return bf16 ? run_tiles<true, 64>(a, f, s) : run_tiles<false, 64>(a, f, s);
}

}  // extern "C"
