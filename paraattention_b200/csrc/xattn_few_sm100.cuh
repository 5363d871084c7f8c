// Cross attention for few query rows: all rows that share a key / value head - group * Sq of them -
// fit 16 (one new token per sequence; a handful of learned queries). There is no reuse to speak
// of, K and V are read once: HBM-bound (latency-bound when the keys are few).
//
// tcgen05 works on 128 rows, of which this shape fills 1 to 16, and its pipeline (TMA, TMEM, five
// hand-overs per key tile) costs microseconds before the first result; mma.sync m16n8k16 fits the
// rows, keeps S, P and O in registers, and at 16 rows its rate is far above what HBM can feed.
//
// One cluster of 1 to 16 CTAs per (batch, kv head), the key tiles of 64 divided among its CTAs,
// so that few heads still fill the GPU in ONE launch: the CTAs' partial results are joined through
// distributed shared memory. Inside a CTA each of 4 warps owns 16 keys of every tile; 4 other warps
// fill a 3-stage cp.async ring with K and V (the copies' addresses and the mask cost as many
// instructions as the arithmetic: one set of warps doing both in turn took 2.6 us per tile with two
// CTAs on an SM, four times what HBM needs). Keys that are masked or behind the last are not
// read: their copy fills zeros (so infinities or NaN there never enter) and their logits are -inf.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "fbc_sm100.cuh"
#include "pa_ptx.cuh"
#include "xattn_sm100.cuh"

namespace pa {

constexpr int kFewRows = 16;
constexpr int kFewKeys = 64;
constexpr int kFewThreads = 128;  // that compute; as many more load
constexpr int kFewStages = 3;  // (6 for CTAs that have an SM to themselves: no faster, the arithmetic is what they wait for)
constexpr int kFewMaxCluster = 16;

struct XFewParams {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    float* lse;
    long long q_s[3], k_s[3], v_s[3], o_s[3];  // element strides (batch, head, row); k_s[0] = 0: one batch entry for all
    const uint8_t* mask;
    long long mask_s;
    int hkv, group, sq, skv;
    float scale, scale_log2;
    int* status;
    int* status_host;
    unsigned long long wait_ns;
};

template <int kD>
constexpr int few_smem_bytes() {
    // Q tile, ring of K and V tiles (reused for the joining), row statistics, barriers
    return kFewRows * kD * 2 + kFewStages * 2 * kFewKeys * kD * 2 + 5 * kFewRows * 8 + 2 * kFewStages * 8 + 16;
}

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool live) {
    const int bytes = live ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <bool kBF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (kBF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool kBF16, int kD>
__global__ void __launch_bounds__(2 * kFewThreads, 2)
xattn_few_kernel(const __grid_constant__ XFewParams p) {
    namespace cg = cooperative_groups;
    constexpr int kChunks = kD / 8;                 // 16-byte chunks of a row
    constexpr int kRowBytes = kD * 2;
    constexpr int kTile = kFewKeys * kRowBytes;     // bytes of a K or V tile
    constexpr int kStage = 2 * kTile;               // K, V
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sq_ = smem;
    uint8_t* ring = smem + kFewRows * kRowBytes;
    float2* wml = reinterpret_cast<float2*>(ring + kFewStages * kStage);  // [4 warps][16 rows]
    float2* cml = wml + 4 * kFewRows;                                     // [16 rows] of this CTA

    uint64_t* full = reinterpret_cast<uint64_t*>(cml + kFewRows);         // [stages], one arrival per loading thread
    uint64_t* empty = full + kFewStages;                                  // [stages], one arrival per computing warp
    int* abort_word = reinterpret_cast<int*>(empty + kFewStages);
    volatile int* s_abort = abort_word;

    auto cluster = cg::this_cluster();
    const int cn = static_cast<int>(cluster.num_blocks()), cr = static_cast<int>(cluster.block_rank());
    const int unit = blockIdx.x / cn;
    const int hk = unit % p.hkv, b = unit / p.hkv;
    const int rows = p.group * p.sq;
    const int tid = threadIdx.x % kFewThreads, lane = tid & 31, warp = tid >> 5;
    const bool loader = threadIdx.x >= kFewThreads;
    const int tiles = (p.skv + kFewKeys - 1) / kFewKeys;
    const int tile0 = static_cast<int>(static_cast<long long>(tiles) * cr / cn);
    const int tile1 = static_cast<int>(static_cast<long long>(tiles) * (cr + 1) / cn);
    const uint8_t* mb = p.mask != nullptr ? p.mask + b * p.mask_s : nullptr;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kFewStages; ++i) {
            mbar_init(smem_u32(full + i), kFewThreads);
            mbar_init(smem_u32(empty + i), kFewThreads / 32);
        }
        *abort_word = 0;
        mbar_init_fence();
    }
    // Q rows: row r = (head r / Sq of the group, query r % Sq); rows that do not exist are zeros
    for (int i = threadIdx.x; i < kFewRows * kChunks; i += 2 * kFewThreads) {
        const int r = i / kChunks, c = i % kChunks;
        const bool live = r < rows;
        const int g = live ? r / p.sq : 0, s = live ? r - g * p.sq : 0;
        const uint16_t* src = p.q + b * p.q_s[0] + (hk * p.group + g) * p.q_s[1] + s * p.q_s[2] + c * 8;
        *reinterpret_cast<uint4*>(sq_ + r * kRowBytes + ((c ^ (r & 7)) << 4)) =
            live ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0, 0, 0, 0);
    }
    __syncthreads();

    if (loader) {
        constexpr int kKeysPerPass = kFewThreads / kChunks, kPasses = kFewKeys / kKeysPerPass;
        const int my_chunk = tid % kChunks, my_key = tid / kChunks;
        const uint16_t* kb = p.k + b * p.k_s[0] + hk * p.k_s[1] + my_chunk * 8;
        const uint16_t* vb = p.v + b * p.v_s[0] + hk * p.v_s[1] + my_chunk * 8;
        for (int t = tile0, n = 0; t < tile1; ++t, ++n) {
            bool keep[kPasses];
#pragma unroll
            for (int i = 0; i < kPasses; ++i) {
                const int key = t * kFewKeys + my_key + i * kKeysPerPass;
                keep[i] = key < p.skv;
                if (mb != nullptr) keep[i] = keep[i] & (__ldg(mb + min(key, p.skv - 1)) != 0);
            }
            const int st = n % kFewStages;
            if (n >= kFewStages &&
                !mbar_wait(smem_u32(empty + st), ((n / kFewStages) & 1) ^ 1, s_abort, p.status, p.wait_ns, PA_DEV_TIMEOUT_PIPE))
                break;
            const uint32_t base = smem_u32(ring + st * kStage);
            const uint16_t* kt = kb + static_cast<long long>(t) * kFewKeys * p.k_s[2];
            const uint16_t* vt = vb + static_cast<long long>(t) * kFewKeys * p.v_s[2];
#pragma unroll
            for (int i = 0; i < kPasses; ++i) {
                const int r = my_key + i * kKeysPerPass;
                const uint32_t at = r * kRowBytes + ((my_chunk ^ (r & 7)) << 4);
                // (a copy of zero bytes reads nothing; its address stays inside the tensor all the same)
                cp_async16_zfill(base + at, keep[i] ? kt + r * p.k_s[2] : kb, keep[i]);
                cp_async16_zfill(base + kTile + at, keep[i] ? vt + r * p.v_s[2] : vb, keep[i]);
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(full + st)) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }

    float o[kChunks][4];
#pragma unroll
    for (int n = 0; n < kChunks; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    uint32_t qa[kD / 16][4];
    const float sl = p.scale_log2;

    // Which of my warp's 16 keys of a tile take part: the byte is looked at a tile ahead.
    auto look = [&](int t) -> uint32_t {
        const int key = t * kFewKeys + warp * 16 + (lane & 15);
        return key < p.skv ? (mb != nullptr ? static_cast<uint32_t>(__ldg(mb + key)) : 1u) : 0u;
    };
    uint32_t next = loader ? 0u : look(tile0);
    if (!loader) {
#pragma unroll
        for (int ks = 0; ks < kD / 16; ++ks) {
            const int r = lane & 15, c = 2 * ks + (lane >> 4);
            ldsm4(smem_u32(sq_ + r * kRowBytes + ((c ^ (r & 7)) << 4)), qa[ks]);
        }
    }
    for (int t = tile0, n = 0; t < tile1 && !loader; ++t, ++n) {
        const uint32_t live = __ballot_sync(0xffffffffu, next != 0) & 0xffffu;
        next = look(t + 1);
        const int slot = n % kFewStages;
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(full + slot), (n / kFewStages) & 1, s_abort, p.status, p.wait_ns, PA_DEV_TIMEOUT_PIPE)))
            break;
        uint8_t* st = ring + slot * kStage;
        if (live == 0) {  // no key of this warp's 16 takes part
            if (lane == 0) mbar_arrive(smem_u32(empty + slot));
            continue;
        }
        float s[2][4];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nb][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < kD / 16; ++ks) {
            const int r = warp * 16 + (lane & 7) + ((lane >> 4) << 3), c = 2 * ks + ((lane >> 3) & 1);
            uint32_t kf[4];
            ldsm4(smem_u32(st + r * kRowBytes + ((c ^ (r & 7)) << 4)), kf);
            mma16816<kBF16>(s[0], qa[ks], kf[0], kf[1]);
            mma16816<kBF16>(s[1], qa[ks], kf[2], kf[3]);
        }
        float mx[2] = {m[0], m[1]};
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int col = nb * 8 + (lane & 3) * 2 + (i & 1);
                s[nb][i] = ((live >> col) & 1u) != 0 ? s[nb][i] * sl : -INFINITY;
                mx[i >> 1] = fmaxf(mx[i >> 1], s[nb][i]);
            }
        float alpha[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
            // (keys that take part may have logits of -inf; 0 is then as good a reference as any)
            const float ref = mx[h] == -INFINITY ? 0.f : mx[h];
            alpha[h] = ex2_approx(m[h] - ref);
            m[h] = mx[h];
            mx[h] = ref;
            l[h] *= alpha[h];
        }
        uint32_t pa_[4];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                e[i] = ex2_approx(s[nb][i] - mx[i >> 1]);
                l[i >> 1] += e[i];
            }
            pa_[2 * nb] = kBF16 ? pack_bf16x2(e[0], e[1]) : pack_f16x2(e[0], e[1]);
            pa_[2 * nb + 1] = kBF16 ? pack_bf16x2(e[2], e[3]) : pack_f16x2(e[2], e[3]);
        }
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
            const int r = warp * 16 + (lane & 15), cc = c + (lane >> 4);
            uint32_t vf[4];
            ldsm4_t(smem_u32(st + kTile + r * kRowBytes + ((cc ^ (r & 7)) << 4)), vf);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[c][i] *= alpha[i >> 1];
                o[c + 1][i] *= alpha[i >> 1];
            }
            mma16816<kBF16>(o[c], pa_, vf[0], vf[1]);
            mma16816<kBF16>(o[c + 1], pa_, vf[2], vf[3]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(empty + slot));
    }
    __syncthreads();
    if (threadIdx.x == 0) x_report(p.status_host, *s_abort);

    // ---- join the 4 warps: O [warp][16][kD] fp32 over the ring ------------------------------------
    float* wo = reinterpret_cast<float*>(ring);
    static_assert(4 * kFewRows * kD * 4 <= kFewStages * kStage, "the ring holds the partial results");
    if (!loader) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        const int r = (lane >> 2) + 8 * h;
        if ((lane & 3) == 0) wml[warp * kFewRows + r] = make_float2(m[h], l[h]);
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
            *reinterpret_cast<float2*>(wo + (warp * kFewRows + r) * kD + c * 8 + (lane & 3) * 2) =
                make_float2(o[c][2 * h], o[c][2 * h + 1]);
    }
    }
    __syncthreads();
    constexpr int kPer = kFewRows * kD / (2 * kFewThreads);  // elements per thread, all of one row
    {
        const int r = threadIdx.x * kPer / kD, c0 = threadIdx.x * kPer % kD;
        float mt = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mt = fmaxf(mt, wml[w * kFewRows + r].x);
        float wgt[4], lt = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float2 ml = wml[w * kFewRows + r];
            wgt[w] = ml.y == 0.f ? 0.f : ex2_approx(ml.x - mt);
            lt += ml.y * wgt[w];
        }
        // (each element is read and written by the same thread)
#pragma unroll
        for (int i = 0; i < kPer; i += 4) {
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float4 x = *reinterpret_cast<const float4*>(wo + (w * kFewRows + r) * kD + c0 + i);
                a.x = fmaf(x.x, wgt[w], a.x);
                a.y = fmaf(x.y, wgt[w], a.y);
                a.z = fmaf(x.z, wgt[w], a.z);
                a.w = fmaf(x.w, wgt[w], a.w);
            }
            *reinterpret_cast<float4*>(wo + r * kD + c0 + i) = a;
        }
        if (c0 == 0) cml[r] = make_float2(mt, lt);
    }
    // ---- join the CTAs of the cluster: 8 output elements per thread -----------------------------------
    if (cn > 1) cluster.sync();
    else __syncthreads();
    for (int i = cr * 2 * kFewThreads + threadIdx.x; i < rows * kChunks; i += cn * 2 * kFewThreads) {
        const int r = i / kChunks, c0 = (i % kChunks) * 8;
        float mt = -INFINITY, lt = 0.f;
        for (int k = 0; k < cn; ++k) mt = fmaxf(mt, cluster.map_shared_rank(cml, k)[r].x);
        float a[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) a[x] = 0.f;
        for (int k = 0; k < cn; ++k) {
            const float2 ml = cluster.map_shared_rank(cml, k)[r];
            if (ml.y == 0.f) continue;  // (saw no key; a sum that is NaN stays one)
            const float wgt = ex2_approx(ml.x - mt);
            lt = fmaf(ml.y, wgt, lt);
            const float4* src = reinterpret_cast<const float4*>(cluster.map_shared_rank(wo, k) + r * kD + c0);
            const float4 x0 = src[0], x1 = src[1];
            a[0] = fmaf(x0.x, wgt, a[0]); a[1] = fmaf(x0.y, wgt, a[1]);
            a[2] = fmaf(x0.z, wgt, a[2]); a[3] = fmaf(x0.w, wgt, a[3]);
            a[4] = fmaf(x1.x, wgt, a[4]); a[5] = fmaf(x1.y, wgt, a[5]);
            a[6] = fmaf(x1.z, wgt, a[6]); a[7] = fmaf(x1.w, wgt, a[7]);
        }
        const float inv = lt != 0.f ? 1.f / lt : 0.f;
        const int g = r / p.sq, s = r - g * p.sq, head = hk * p.group + g;
        uint32_t w[4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
            w[x] = kBF16 ? pack_bf16x2(a[2 * x] * inv, a[2 * x + 1] * inv) : pack_f16x2(a[2 * x] * inv, a[2 * x + 1] * inv);
        *reinterpret_cast<uint4*>(p.out + b * p.o_s[0] + head * p.o_s[1] + s * p.o_s[2] + c0) = make_uint4(w[0], w[1], w[2], w[3]);
        if (c0 == 0 && p.lse != nullptr)
            p.lse[(static_cast<long long>(b) * p.hkv * p.group + head) * p.sq + s] =
                lt != 0.f ? 0.6931471805599453f * (mt + log2f(lt)) : -INFINITY;
    }
    if (cn > 1) cluster.sync();  // (nobody leaves while its shared memory is still read)
}

}  // namespace pa
