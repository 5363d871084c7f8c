// C ABI of cross attention, backward: argument validation and launches.
#include "pa_xattn_host.h"
#include "xattn_bwd_sm100.cuh"

using namespace pa_host;

namespace {

struct BwdPlan {
    pa::XSched q, k;  // query pass, key pass
    int grid_q = 0, grid_k = 0, mt = 0, kt = 0;
    int bound_parts = 0, bound_keys = 0;  // f16: parts of a key head's values and their keys (a multiple of 64)
    int64_t off_stats = 0, off_do_max = 0, off_v_max = 0, off_part = 0, bytes = 0;
};

BwdPlan plan(const pa_xattn_args* a) {
    BwdPlan f;
    f.mt = (a->seq_q + 127) / 128;
    f.kt = (a->seq_kv + 127) / 128;
    const int sms = sm_count();
    f.q = xattn_schedule(static_cast<long long>(a->batch) * a->heads * f.mt, f.kt, 1, sms, 4, &f.grid_q);
    f.k = xattn_schedule(static_cast<long long>(a->kv_batch) * a->kv_heads * f.kt,
                         static_cast<long long>(a->batch / a->kv_batch) * (a->heads / a->kv_heads) * f.mt, f.kt, sms, 4, &f.grid_k);
    f.off_stats = xattn_mask_layout(a).bytes;
    f.off_part = f.off_stats + int64_t(a->batch) * a->heads * f.mt * 128 * 8;
    if (a->dtype == PA_F16) {
        const int64_t shared = int64_t(a->kv_batch) * a->kv_heads;
        f.bound_keys = ((a->seq_kv + pa::kXBoundParts - 1) / pa::kXBoundParts + 63) / 64 * 64;
        f.bound_parts = (a->seq_kv + f.bound_keys - 1) / f.bound_keys;
        f.off_do_max = f.off_part;
        f.off_v_max = f.off_do_max + up256(shared * 4);
        f.off_part = f.off_v_max + up256(shared * pa::kXBoundParts * 4);
    }
    // (the passes run one after the other and use the same partial results' space)
    const int64_t slots = std::max(f.q.split ? 2 * f.grid_q : 0, f.k.split ? 2 * f.grid_k : 0);
    f.bytes = f.off_part + slots * 2 * 128 * a->head_dim * 4;
    return f;
}

template <bool kBF16, int kD, bool kKeys>
int pass(const CUtensorMap& x, const CUtensorMap& y, const CUtensorMap& z, const CUtensorMap& w, const CUtensorMap& g0,
         const CUtensorMap& g1, const pa::XBwdParams& p, int grid, cudaStream_t s) {
    auto kern = pa::xattn_bwd_kernel<kBF16, kD, kKeys>;
    int rc = allow_smem(kern, pa::kXBwdSmemBytes, "xattn backward");
    if (rc != PA_OK) return rc;
    kern<<<grid, pa::kXBwdThreads, pa::kXBwdSmemBytes, s>>>(x, y, z, w, g0, g1, p);
    rc = launched("xattn backward");
    if (rc != PA_OK || !p.sched.split) return rc;
    pa::XCutList cuts;
    pa::x_list_cuts(p.sched, grid, &cuts);
    if (cuts.n == 0) return PA_OK;
    pa::xattn_bwd_join_kernel<kBF16, kD, kKeys><<<dim3(cuts.n, kD / 8, kKeys ? 2 : 1), 128, 0, s>>>(p, cuts);
    return launched("xattn backward join");
}

template <bool kBF16, int kD>
int run(const pa_xattn_args* a, const BwdPlan& f, cudaStream_t s) {
    CUtensorMap mq, mk, mv, mg, mo, mdq, mdk, mdv;  // (boxes of 128 x 64 for loads, 32 x 32 for stores)
    int rc = make_map(&mq, a->q, a->dtype, kD, a->seq_q, a->heads, a->batch, 1, a->q_stride[2], a->q_stride[1], a->q_stride[0], 0, "q");
    if (rc == PA_OK) rc = make_map(&mg, a->dout, a->dtype, kD, a->seq_q, a->heads, a->batch, 1, a->do_stride[2], a->do_stride[1], a->do_stride[0], 0, "dout");
    if (rc == PA_OK) rc = make_map(&mk, a->k, a->dtype, kD, a->seq_kv, a->kv_heads, a->kv_batch, 1, a->k_stride[2], a->k_stride[1], a->k_stride[0], 0, "k");
    if (rc == PA_OK) rc = make_map(&mv, a->v, a->dtype, kD, a->seq_kv, a->kv_heads, a->kv_batch, 1, a->v_stride[2], a->v_stride[1], a->v_stride[0], 0, "v");
    const bool queries = a->dq != nullptr, keys = a->dk != nullptr;
    if (rc == PA_OK && queries) rc = make_map(&mo, a->out, a->dtype, kD, a->seq_q, a->heads, a->batch, 1, a->o_stride[2], a->o_stride[1], a->o_stride[0], 0, "out");
    if (rc == PA_OK && queries) rc = make_map(&mdq, a->dq, a->dtype, kD, a->seq_q, a->heads, a->batch, 1, a->dq_stride[2], a->dq_stride[1], a->dq_stride[0], 0, "dq", 32, 32);
    if (rc == PA_OK && keys) rc = make_map(&mdk, a->dk, a->dtype, kD, a->seq_kv, a->kv_heads, a->kv_batch, 1, a->dk_stride[2], a->dk_stride[1], a->dk_stride[0], 0, "dk", 32, 32);
    if (rc == PA_OK && keys) rc = make_map(&mdv, a->dv, a->dtype, kD, a->seq_kv, a->kv_heads, a->kv_batch, 1, a->dv_stride[2], a->dv_stride[1], a->dv_stride[0], 0, "dv", 32, 32);
    if (rc != PA_OK) return rc;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    pa::XBwdParams p;
    memset(&p, 0, sizeof(p));
    p.kv_batch = a->kv_batch;
    p.hkv = a->kv_heads;
    p.group = a->heads / a->kv_heads;
    p.sq = a->seq_q;
    p.skv = a->seq_kv;
    p.mt = f.mt;
    p.scale = a->scale;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.by_group = pa::x_div(p.group);
    p.by_mt = pa::x_div(f.mt);
    p.by_b_steps = pa::x_div(p.group * f.mt);
    p.stats = reinterpret_cast<float*>(ws + f.off_stats);
    p.part = reinterpret_cast<float*>(ws + f.off_part);
    p.status = a->status;
    p.status_host = a->status_host;
    p.wait_ns = a->wait_limit_ns ? a->wait_limit_ns : 2000000000ull;
    if (a->key_mask != nullptr) {
        p.words = reinterpret_cast<unsigned long long*>(ws);
        p.extent = reinterpret_cast<int*>(ws + xattn_mask_layout(a).words_bytes);
        pa::xattn_mask_kernel<<<a->batch, pa::kXMaskThreads, 0, s>>>(a->key_mask, a->mask_stride, a->seq_kv,
                                                                     reinterpret_cast<unsigned long long*>(ws),
                                                                     const_cast<int*>(p.extent));
        rc = launched("xattn mask");
        if (rc != PA_OK) return rc;
    }
    if constexpr (!kBF16) {
        pa::XBoundParams bp;
        memset(&bp, 0, sizeof(bp));
        bp.v = static_cast<const uint16_t*>(a->v);
        for (int i = 0; i < 3; ++i) bp.v_s[i] = a->v_stride[i];
        bp.words = p.words;
        bp.batch = a->batch;
        bp.kv_batch = a->kv_batch;
        bp.hkv = a->kv_heads;
        bp.skv = a->seq_kv;
        bp.keys = f.bound_keys;
        bp.v_max = reinterpret_cast<unsigned*>(ws + f.off_v_max);
        bp.do_max = reinterpret_cast<unsigned*>(ws + f.off_do_max);
        p.v_max = bp.v_max;
        p.do_max = bp.do_max;
        p.v_parts = f.bound_parts;
        pa::xattn_bound_kernel<kD><<<dim3(a->kv_batch * a->kv_heads, f.bound_parts), pa::kXBoundThreads, 0, s>>>(bp);
        rc = launched("xattn bounds");
        if (rc != PA_OK) return rc;
    }
    if (queries) {
        pa::XBwdParams pq = p;
        pq.sched = f.q;
        pq.by_tiles = pa::x_div(f.mt);
        pq.by_heads = pa::x_div(a->heads);
        pq.o = static_cast<const uint16_t*>(a->out);
        for (int i = 0; i < 3; ++i) pq.o_s[i] = a->o_stride[i];
        pq.lse = a->lse;
        pq.g[0] = static_cast<uint16_t*>(a->dq);
        pq.g_sb[0] = a->dq_stride[0]; pq.g_sh[0] = a->dq_stride[1]; pq.g_ss[0] = a->dq_stride[2];
        rc = pass<kBF16, kD, false>(mq, mg, mk, mv, mdq, mo, pq, f.grid_q, s);
        if (rc != PA_OK || !keys) return rc;
    } else {
        pa::XStatParams st;
        memset(&st, 0, sizeof(st));
        st.o = static_cast<const uint16_t*>(a->out);
        st.g = static_cast<const uint16_t*>(a->dout);
        for (int i = 0; i < 3; ++i) {
            st.o_s[i] = a->o_stride[i];
            st.g_s[i] = a->do_stride[i];
        }
        st.lse = a->lse;
        st.stats = p.stats;
        st.batch = a->batch;
        st.heads = a->heads;
        st.sq = a->seq_q;
        st.padded = f.mt * 128;
        st.do_max = p.do_max;
        st.kv_batch = a->kv_batch;
        st.hkv = a->kv_heads;
        st.by_group = p.by_group;
        const long long vectors = static_cast<long long>(a->batch) * a->heads * st.padded, per_cta = pa::kXStatThreads / (kD / 8) * 4;
        const int stat_grid = static_cast<int>(std::min<long long>((vectors + per_cta - 1) / per_cta, 8ll * sm_count()));
        pa::xattn_stat_kernel<kBF16, kD><<<stat_grid, pa::kXStatThreads, 0, s>>>(st);
        rc = launched("xattn row statistics");
        if (rc != PA_OK) return rc;
    }
    p.sched = f.k;
    p.by_tiles = pa::x_div(f.kt);
    p.by_heads = pa::x_div(a->kv_heads);
    p.g[0] = static_cast<uint16_t*>(a->dk);
    p.g[1] = static_cast<uint16_t*>(a->dv);
    p.g_sb[0] = a->dk_stride[0]; p.g_sh[0] = a->dk_stride[1]; p.g_ss[0] = a->dk_stride[2];
    p.g_sb[1] = a->dv_stride[0]; p.g_sh[1] = a->dv_stride[1]; p.g_ss[1] = a->dv_stride[2];
    return pass<kBF16, kD, true>(mk, mv, mq, mg, mdk, mdv, p, f.grid_k, s);
}

}  // namespace

extern "C" {

int64_t pa_xattn_bwd_workspace_bytes_(const pa_xattn_args* a) { return plan(a).bytes; }

int pa_xattn_bwd(const pa_xattn_args* a, void* stream) {
    int rc = xattn_sizes(a);
    if (rc == PA_OK) rc = xattn_tensor(a->q, a->q_stride, "q");
    if (rc == PA_OK) rc = xattn_tensor(a->k, a->k_stride, "k");
    if (rc == PA_OK) rc = xattn_tensor(a->v, a->v_stride, "v");
    if (rc == PA_OK) rc = xattn_tensor(a->out, a->o_stride, "out");
    if (rc == PA_OK) rc = xattn_tensor(a->dout, a->do_stride, "dout");
    if (rc == PA_OK && a->dq != nullptr) rc = xattn_tensor(a->dq, a->dq_stride, "dq");
    if (rc == PA_OK && a->dk != nullptr) rc = xattn_tensor(a->dk, a->dk_stride, "dk");
    if (rc == PA_OK && a->dk != nullptr) rc = xattn_tensor(a->dv, a->dv_stride, "dv");
    if (rc != PA_OK) return rc;
    if (a->dk == nullptr && (a->dv != nullptr || a->dq == nullptr))
        return fail(PA_EINVAL, "xattn: the backward call computes dq, or dk and dv, or all three");
    if (a->lse == nullptr) return fail(PA_EINVAL, "xattn: the backward call needs the forward call's lse");
    const BwdPlan f = plan(a);
    if (a->workspace == nullptr || (reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0 || a->workspace_bytes < f.bytes)
        return fail(PA_EINVAL, "xattn: needs a 256-byte aligned workspace of %lld bytes", static_cast<long long>(f.bytes));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf16 = a->dtype == PA_BF16;
    if (a->head_dim == 128) return bf16 ? run<true, 128>(a, f, s) : run<false, 128>(a, f, s);
    return bf16 ? run<true, 64>(a, f, s) : run<false, 64>(a, f, s);
}

}  // extern "C"
