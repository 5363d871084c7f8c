// Cross attention backward for B200. With P = exp(s q k^T - lse), delta = rowsum(do * out):
//   dP = do v^T,  dS = P * (dP - delta),  dq = s dS k,  dk = s dS^T q,  dv = P^T do.
//
// Two passes of ONE kernel: the query pass (kKeys = false) owns tiles of 128 query rows and walks
// the keys for dq; the key pass (kKeys = true) owns tiles of 128 keys and walks the queries (of every
// head that shares the key head, and of every batch entry that shares the keys) for dk and dv. In
// both, the owned pair (X, Y) = (q, do) or (k, v) stays on the SM, the other pair (Z, W) = (k, v) or
// (q, do) streams through rings in tiles of 128 rows, one tile a step, and per step
//   T1 = X Z^T, T2 = Y W^T                (tensor core, 128 x 128, into TMEM)
//   P = 2^(T1 sl - lse'), dS = P (T2 - delta)   (one thread per owned row and 32 columns)
//   A1 += dS Z  [, A2 += P W in the key pass]   (tensor core, dS and P as TMEM operands)
// so dS and P never leave TMEM and are never transposed: the key pass computes their transposes
// to begin with. The price is that S and dP are computed twice (7 products instead of 5); what it
// buys is no atomics (sums in a fixed order), no fp32 dq traffic, and each gradient written once.
//
// The two products of a step form two chains that hide each other's elementwise phases:
//   key pass:    A2(j) T1(j+1) | A1(j) T2(j+1) | ...    P(j+1) is made while A1(j), T2(j+1) run,
//                                                       dS(j+1) while A2(j+1), T1(j+2) run
//   query pass:  T1(j+1) A1(j) T2(j+1) | ...            P is not an operand: T1(j+1) starts as soon as
//                                                       T1(j) has been read
// Measured on the way (16380 queries x 512 keys x 40 heads, cycles per 128 rows, key pass): two chains
// over half tiles (N = 64 products) 4600 with 8 elementwise warps and a two-stage ring, the tensor
// core waiting 1600 of them for loads; 4200 with 16 warps and a finer ring, bound by the issue and the
// operand fetch of the N = 64 products (66 cycles each instead of 32). Whole tiles halve the number of
// products and their shared-memory traffic per flop: the bound is 2048 cycles of products (64 per
// 128 x 128 x 16) and as many of shared memory. The query pass holds X and Y in TMEM, where A2 is not
// needed, and fetches only Z and W from shared memory.
//
// Warps 0-15 elementwise (32 columns each), 16 MMA issuer, 17 TMA producer, 18 clears masked rows of
// K. TMEM columns: T1 [0,128), T2 [128,256), A1 [256, 256 + D), A2 [256 + D, 256 + 2 D) or X, Y [384,
// 512); dS overwrites T2, P overwrites T1. CTAs are persistent and the roles run ahead across units
// (xattn_sm100.cuh divides the work).
//
// What is rounded: P and dS to the tensors' 16-bit type, as operands of a 16-bit product (their
// relative error, half an ulp, averages out over the sum); everything else is fp32. bf16 has fp32's range. f16
// has not: below 2^-14 its steps are 2^-24, whatever the value, and dS, about |do| / Skv times ten, is there for
// ordinary gradients (8192 keys, do of 1e-3: dq off by 7.6e-3 of itself); above 65504 it is infinite. So in f16 both
// are powers of two larger or smaller than they are, and the epilogue takes that back, exactly, from the fp32 sums:
//   P by 2^14 (P <= 1);
//   dS by 2^e with |dS| 2^e < 2^15. |dS| <= P (|dP| + |delta|) <= 2 sum|do| max|v|, since out is an average of values;
//     sum over a row of do, max over the values of the key head that take part. The query pass has an e of its own for
//     each row; the key pass, which adds up over rows, has the one of the key head's largest row.
// max|v| comes from a launch in front (xattn_bound_kernel), sum|do| from where the row statistics are made. What is
// not finite takes no part in the bounds: it makes its own results so, and no other's. The half steps of dS are then at
// most 2^-39 of that bound. (Masked values take no part either: they may hold anything.)
#pragma once
#include <type_traits>

#include "fbc_sm100.cuh"
#include "xattn_sm100.cuh"

namespace pa {

constexpr int kXBwdSoftWarps = 16;
constexpr int kXBwdMmaWarp = 16, kXBwdTmaWarp = 17, kXBwdCleanWarp = 18;
constexpr int kXBwdThreads = 640;
// Z is needed from T1 to A1, W from T2 to A2 or less: three stages of Z and two of W leave every load
// the time of five products.
constexpr int kXZStages = 3, kXWStages = 2;
// f16: the exponent of P, and how many parts of a key head's values the launch in front of the passes bounds by themselves.
constexpr int kXShiftP = 14;
constexpr int kXBoundParts = 32;

struct XBwdParams {
    int kv_batch, hkv, group, sq, skv;
    int mt;           // 128-row tiles of the queries
    float scale, scale_log2;
    uint16_t* g[2];   // query pass: dq, -; key pass: dk, dv (written with TMA, but for joined or empty tiles)
    long long g_sb[2], g_sh[2], g_ss[2];
    // [B][Hq][mt][-lse * log2 e (f16: + kXShiftP), -delta][128 rows]; rows behind the last query, and rows without
    // any key, have (-inf, 0), which makes their P zero. Read by the key pass; written by the query pass if
    // there is one, which has do on the SM anyway (97 us more for it, against 122 us for a kernel of its own, at
    // 32760 x 512 x 40 heads; 8 against 14 us at 2 x 2049 x 333 x 32 heads), else by xattn_stat_kernel.
    float* stats;
    const uint16_t* o;  // query pass: out
    long long o_s[3];
    const float* lse;   // query pass: [B][Hq][Sq]
    // f16: per [kv batch][kv head], the largest |v| of each part of its keys and the largest sum|do| of a row of its
    // queries (float bits; written by the query pass or xattn_stat_kernel, read by the key pass)
    const unsigned* v_max;  // [][kXBoundParts], the first v_parts written
    unsigned* do_max;
    int v_parts;
    const unsigned long long* words;
    const int* extent;
    XSched sched;
    XDiv by_tiles, by_heads;           // of the owned tensors
    XDiv by_group, by_mt, by_b_steps;  // by_b_steps: the key pass's steps of a batch entry
    float* part;      // [slot][A1, A2][D / 4][128 rows][4]
    int* status;
    int* status_host;
    unsigned long long wait_ns;
};

struct XBwdCtl {
    uint64_t xy_full, xy_empty;
    uint64_t xt_full;               // query pass: X and Y are in TMEM (one arrival per warp)
    uint64_t stat_full;             // query pass: lse and do * out of the owned rows are in `stat` (one arrival per warp)
    uint64_t z_full[kXZStages], z_empty[kXZStages], z_clean[kXZStages];
    uint64_t w_full[kXWStages], w_empty[kXWStages];
    uint64_t t1_full, t2_full;
    uint64_t p_full;                // key pass: P is in TMEM; query pass: T1 has been read (one arrival per warp)
    uint64_t ds_full;               // dS is in TMEM (one arrival per warp)
    uint64_t acc_done;              // A1, A2 of a segment are complete
    uint64_t acc_free;              // the epilogue has read them (one arrival per warp)
    uint64_t teardown;
    uint32_t tmem_base;
    int abort;
};
// Operands, row statistics, control block. (The dynamic shared memory is declared with the
// alignment of the swizzle; there is no room for slack.)
constexpr int kXBwdStatBytes = kXWStages * kTileN * 8;
constexpr int kXBwdSmemBytes = (2 + kXZStages + kXWStages) * kTileBytes + kXBwdStatBytes + 512;
static_assert(sizeof(XBwdCtl) <= 512, "control block too large");
static_assert(kXBwdSmemBytes <= 232448, "shared memory");

// Where a segment's owned tile and a step's streamed tile lie.
struct XBwdUnit {
    int b, head, tile;  // owned tile: batch entry (of its tensor), head (of its tensor), 128-row tile
    int t0, t1;
};
struct XBwdStep {
    int b, head, tile;  // streamed tile
};

template <bool kKeys>
__device__ __forceinline__ XBwdUnit x_bwd_unit(const XBwdParams& p, const XSeg& g) {
    XBwdUnit u;
    const int x = p.by_tiles(g.unit);
    u.tile = g.unit - x * static_cast<int>(p.by_tiles.d);
    u.b = p.by_heads(x);
    u.head = x - u.b * static_cast<int>(p.by_heads.d);
    u.t0 = g.t0;
    u.t1 = g.t1;
    if (!kKeys && p.extent != nullptr) {  // key tiles behind the last key that takes part
        const int n = (__ldg(p.extent + u.b) + kTileN - 1) / kTileN;
        u.t1 = min(u.t1, n);
        u.t0 = min(u.t0, u.t1);
    }
    return u;
}
// Key pass: steps run over (batch entries that share the keys, heads of the group, query tiles).
template <bool kKeys>
__device__ __forceinline__ XBwdStep x_bwd_step(const XBwdParams& p, const XBwdUnit& u, int step) {
    XBwdStep s;
    if (!kKeys) {
        s.b = p.kv_batch == 1 ? 0 : u.b;
        s.head = p.by_group(u.head);
        s.tile = step;
        return s;
    }
    const int m = p.by_mt(step);
    s.tile = step - m * p.mt;
    const int bb = p.by_group(m);
    s.head = u.head * p.group + (m - bb * p.group);
    s.b = p.kv_batch == 1 ? bb : u.b;
    return s;
}
// The first step >= `step` with something to do (the segment's end if none): the key pass skips batch
// entries whose mask ends before the owned keys.
template <bool kKeys>
__device__ __forceinline__ int x_bwd_live(const XBwdParams& p, const XBwdUnit& u, int step) {
    if (!kKeys || p.extent == nullptr) return step;
    const int per_b = p.group * p.mt;
    while (step < u.t1) {
        const int b = p.kv_batch == 1 ? p.by_b_steps(step) : u.b;
        if (u.tile * kTileN < __ldg(p.extent + b)) return step;
        if (p.kv_batch != 1) return u.t1;
        step = (b + 1) * per_b;
    }
    return u.t1;
}
// The unit of the next segment that has steps, if any.
template <bool kKeys>
__device__ __forceinline__ bool x_bwd_more(const XBwdParams& p, XCursor cursor, XBwdUnit& u) {
    XSeg g;
    while (cursor.next(p.sched, g)) {
        u = x_bwd_unit<kKeys>(p, g);
        if (x_bwd_live<kKeys>(p, u, u.t0) < u.t1) return true;
    }
    return false;
}

// Sum of the products of two chunks of 8 elements.
template <bool kBF16>
__device__ __forceinline__ float dot8(const uint32_t* x, const uint32_t* y) {
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        dot = fmaf(lo16<kBF16>(x[i]), lo16<kBF16>(y[i]), dot);
        dot = fmaf(hi16<kBF16>(x[i]), hi16<kBF16>(y[i]), dot);
    }
    return dot;
}

// Sum of the magnitudes of a chunk of 8 elements.
template <bool kBF16>
__device__ __forceinline__ float abs8(const uint32_t* x) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += fabsf(lo16<kBF16>(x[i])) + fabsf(hi16<kBF16>(x[i]));
    return sum;
}
// f16: the exponent e with 2 bound 2^e in [2^14, 2^15) (bound: a product of sums and values of f16 numbers, so 2^-48
// to 2^40 if it is finite and not zero), and 2^-e.
__device__ __forceinline__ int x_slope_exp(float bound) {
    return bound > 0.f && bound < INFINITY ? 13 - (static_cast<int>(__float_as_uint(bound) >> 23) - 127) : 0;
}
__device__ __forceinline__ float x_pow2(int e) { return __uint_as_float(static_cast<unsigned>(127 + e) << 23); }
// The largest |v| of a (kv batch, kv head). A whole warp calls.
__device__ __forceinline__ float x_v_max(const XBwdParams& p, int unit, int lane) {
    const unsigned m = lane < p.v_parts ? __ldg(p.v_max + static_cast<long long>(unit) * kXBoundParts + lane) : 0u;
    return __uint_as_float(__reduce_max_sync(0xffffffffu, m));
}

template <bool kBF16, int kD, bool kKeys>
__global__ void __launch_bounds__(kXBwdThreads, 1)
xattn_bwd_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_y,
                 const __grid_constant__ CUtensorMap tm_z, const __grid_constant__ CUtensorMap tm_w,
                 const __grid_constant__ CUtensorMap tm_g0, const __grid_constant__ CUtensorMap tm_g1,
                 const __grid_constant__ XBwdParams p) {
    constexpr int kAtoms = kD / 64;
    constexpr int kOperandBytes = kAtoms * kHalfBytes;
    constexpr uint32_t kColT1 = 0, kColT2 = 128, kColA1 = 256, kColA2 = 256 + kD;
    constexpr uint32_t kColX = 384, kColY = 448;  // query pass
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sX = smem_u32(smem), sY = sX + kTileBytes, sZ = sX + 2 * kTileBytes, sW = sZ + kXZStages * kTileBytes;
    uint8_t* smem_z = smem + 2 * kTileBytes;
    // key pass: [W stage][2][128], a step's row statistics; query pass: [3][128], lse and do * out of the owned rows and,
    // in f16, the exponent of their dS
    float* stat = reinterpret_cast<float*>(smem + (2 + kXZStages + kXWStages) * kTileBytes);
    XBwdCtl* ctl = reinterpret_cast<XBwdCtl*>(smem + (2 + kXZStages + kXWStages) * kTileBytes + kXBwdStatBytes);
    volatile int* s_abort = &ctl->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        int st = p.status != nullptr ? *reinterpret_cast<volatile int*>(p.status) : 0;
        if ((sX & 1023u) != 0) {  // (never seen; the swizzled tiles would not be where the descriptors say)
            st = PA_DEV_TIMEOUT_PIPE;
            if (p.status != nullptr) atomicCAS(p.status, 0, st);
        }
        x_report(p.status_host, st);  // (a launch that does nothing because of an earlier one's wait says so, too)
        ctl->abort = st;
    }
    __syncthreads();
    if (ctl->abort != 0) return;
    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&ctl->xy_full), 1);
        mbar_init(smem_u32(&ctl->xy_empty), kXBwdSoftWarps);
        mbar_init(smem_u32(&ctl->xt_full), kXBwdSoftWarps);
        mbar_init(smem_u32(&ctl->stat_full), kXBwdSoftWarps);
        for (int s = 0; s < kXZStages; ++s) {
            mbar_init(smem_u32(&ctl->z_full[s]), 1);
            mbar_init(smem_u32(&ctl->z_empty[s]), 1);
            mbar_init(smem_u32(&ctl->z_clean[s]), 1);
        }
        for (int s = 0; s < kXWStages; ++s) {
            mbar_init(smem_u32(&ctl->w_full[s]), 1);
            // (the key pass's statistics share the stage: the warps that read them arrive too)
            mbar_init(smem_u32(&ctl->w_empty[s]), kKeys ? 1 + kXBwdSoftWarps : 1);
        }
        mbar_init(smem_u32(&ctl->t1_full), 1);
        mbar_init(smem_u32(&ctl->t2_full), 1);
        mbar_init(smem_u32(&ctl->p_full), kXBwdSoftWarps);
        mbar_init(smem_u32(&ctl->ds_full), kXBwdSoftWarps);
        mbar_init(smem_u32(&ctl->acc_done), 1);
        mbar_init(smem_u32(&ctl->acc_free), kXBwdSoftWarps);
        mbar_init(smem_u32(&ctl->teardown), 1);
        mbar_init_fence();
    }
    if (warp == kXBwdMmaWarp) {
        tmem_alloc(smem_u32(&ctl->tmem_base), kTmemCols);
        tmem_relinquish();
    }
    if (warp == kXBwdTmaWarp && lane == 0) {
        tma_prefetch_desc(&tm_x);
        tma_prefetch_desc(&tm_y);
        tma_prefetch_desc(&tm_z);
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_g0);
        if (kKeys) tma_prefetch_desc(&tm_g1);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;
    const uint64_t limit = p.wait_ns;
    const int n_words = (p.skv + 63) >> 6;
    const bool clean = !kKeys && p.words != nullptr;  // masked rows of K are zeroed before use

    XCursor cursor(p.sched);
    XSeg seg;
    if (warp == kXBwdTmaWarp) {
        // =============================== TMA producer ======================================
        if (lane == 0) {
            auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
                return mbar_wait(smem_u32(bar), parity, s_abort, p.status, limit, PA_DEV_TIMEOUT_PIPE);
            };
            bool ok = true;
            int j = 0, n_seg = 0;
            while (ok && cursor.next(p.sched, seg)) {
                const XBwdUnit u = x_bwd_unit<kKeys>(p, seg);
                int st = x_bwd_live<kKeys>(p, u, u.t0);
                if (st >= u.t1) continue;
                if (n_seg > 0) ok = wait(&ctl->xy_empty, (n_seg - 1) & 1);
                if (!ok) break;
                const uint32_t bx = smem_u32(&ctl->xy_full);
                mbar_expect_tx(bx, 2 * kOperandBytes);
#pragma unroll
                for (int h = 0; h < kAtoms; ++h) {
                    tma_load_5d(sX + h * kHalfBytes, &tm_x, bx, h * 64, u.tile * kTileM, u.head, u.b, 0);
                    tma_load_5d(sY + h * kHalfBytes, &tm_y, bx, h * 64, u.tile * kTileM, u.head, u.b, 0);
                    if (!kKeys) tma_prefetch_5d(&tm_g1, h * 64, u.tile * kTileM, u.head, u.b, 0);  // (out)
                }
                for (; st < u.t1; st = x_bwd_live<kKeys>(p, u, st + 1), ++j) {
                    const XBwdStep s = x_bwd_step<kKeys>(p, u, st);
                    const int zs = j % kXZStages, ws = j % kXWStages;
                    if (j >= kXZStages) ok = wait(&ctl->z_empty[zs], ((j / kXZStages) & 1) ^ 1);
                    if (!ok) break;
                    const uint32_t bz = smem_u32(&ctl->z_full[zs]);
                    mbar_expect_tx(bz, kOperandBytes);
#pragma unroll
                    for (int h = 0; h < kAtoms; ++h)
                        tma_load_5d(sZ + zs * kTileBytes + h * kHalfBytes, &tm_z, bz, h * 64, s.tile * kTileN, s.head, s.b, 0);
                    if (j >= kXWStages) ok = wait(&ctl->w_empty[ws], ((j / kXWStages) & 1) ^ 1);
                    if (!ok) break;
                    const uint32_t bw = smem_u32(&ctl->w_full[ws]);
                    mbar_expect_tx(bw, kOperandBytes + (kKeys ? kTileN * 8 : 0));
#pragma unroll
                    for (int h = 0; h < kAtoms; ++h)
                        tma_load_5d(sW + ws * kTileBytes + h * kHalfBytes, &tm_w, bw, h * 64, s.tile * kTileN, s.head, s.b, 0);
                    if (kKeys) {
                        const float* src = p.stats + ((static_cast<long long>(s.b) * p.hkv * p.group + s.head) * p.mt + s.tile) * (2 * kTileN);
                        asm volatile(
                            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                smem_u32(stat + ws * 2 * kTileN)),
                            "l"(src), "r"(kTileN * 8), "r"(bw)
                            : "memory");
                    }
                }
                ++n_seg;
            }
            if (*s_abort != 0) {  // leave only once copies already issued have landed (bounded)
                int none = 0;
                volatile int* no_abort = &none;
                if (n_seg > 0) mbar_wait(smem_u32(&ctl->xy_full), (n_seg - 1) & 1, no_abort, nullptr, 10000000ull, 0);
                mbar_wait(smem_u32(&ctl->xy_full), n_seg & 1, no_abort, nullptr, 10000000ull, 0);
                for (int jj = (j > kXZStages ? j - kXZStages : 0); jj <= j; ++jj) {
                    mbar_wait(smem_u32(&ctl->z_full[jj % kXZStages]), (jj / kXZStages) & 1, no_abort, nullptr, 10000000ull, 0);
                    mbar_wait(smem_u32(&ctl->w_full[jj % kXWStages]), (jj / kXWStages) & 1, no_abort, nullptr, 10000000ull, 0);
                }
            }
        }
    } else if (warp == kXBwdMmaWarp) {
        // =============================== MMA issuer ========================================
        constexpr uint32_t idesc_t = make_idesc_f16(kBF16, false, kTileM, kTileN);
        constexpr uint32_t idesc_a = make_idesc_f16(kBF16, true, kTileM, kD);
        const uint32_t leader = elect_one() ? 1u : 0u;
        // K-major descriptors (T1, T2) and MN-major descriptors (the same tiles as B operands of A1, A2)
        const uint64_t dk0 = smem_desc_sw128(sX, 16, 1024), dm0 = smem_desc_sw128(sZ, kHalfBytes, 1024);
        const uint32_t hi_k = static_cast<uint32_t>(dk0 >> 32), hi_m = static_cast<uint32_t>(dm0 >> 32);
        const uint32_t lo_x = static_cast<uint32_t>(dk0), lo_y = lo_x + (kTileBytes >> 4);
        const uint32_t lo_z = static_cast<uint32_t>(smem_desc_sw128(sZ, 16, 1024)), lo_w = lo_z + (kXZStages * kTileBytes >> 4);
        const uint32_t lo_zm = static_cast<uint32_t>(dm0), lo_wm = lo_zm + (kXZStages * kTileBytes >> 4);
        auto issue_t = [&](uint32_t lo_own, uint32_t col_own, uint32_t lo_b, uint32_t col, uint64_t* full) {
#pragma unroll
            for (int ks = 0; ks < kD / 16; ++ks) {
                const uint32_t off = ((ks >> 2) * kHalfBytes + (ks & 3) * 32) >> 4;
                if (kKeys) tc_mma_ss_elect(tmem + col, lo_own + off, hi_k, lo_b + off, hi_k, idesc_t, ks > 0 ? 1u : 0u, leader);
                else tc_mma_ts_elect(tmem + col, tmem + col_own + ks * 8, lo_b + off, hi_k, idesc_t, ks > 0 ? 1u : 0u, leader);
            }
            tc_commit_elect(smem_u32(full), leader);
        };
        auto issue_t1 = [&](int j) { issue_t(lo_x, kColX, lo_z + ((j % kXZStages) * kTileBytes >> 4), kColT1, &ctl->t1_full); };
        auto issue_t2 = [&](int j) {
            issue_t(lo_y, kColY, lo_w + ((j % kXWStages) * kTileBytes >> 4), kColT2, &ctl->t2_full);
            if (!kKeys) tc_commit_elect(smem_u32(&ctl->w_empty[j % kXWStages]), leader);
        };
        // 16 streamed rows a k-step; their dS / P are 8 packed columns (32 columns of T are packed into 16)
        auto issue_a = [&](uint32_t col_a, uint32_t col_t, uint32_t lo_b, bool acc) {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
                tc_mma_ts_elect(tmem + col_a, tmem + col_t + (ks >> 1) * 32 + (ks & 1) * 8, lo_b + ((ks * 16 * 128) >> 4), hi_m, idesc_a,
                                (acc || ks > 0) ? 1u : 0u, leader);
        };
        auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
            const bool r = __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, s_abort, p.status, limit, PA_DEV_TIMEOUT_PIPE));
            tc_fence_after();
            return r;
        };
        auto wait_z = [&](int j) -> bool {
            return wait(clean ? &ctl->z_clean[j % kXZStages] : &ctl->z_full[j % kXZStages], (j / kXZStages) & 1);
        };
        auto wait_w = [&](int j) -> bool { return wait(&ctl->w_full[j % kXWStages], (j / kXWStages) & 1); };
        bool ok = true, issued = false;
        int j = 0, n_seg = 0;  // steps, segments with steps
        while (ok && cursor.next(p.sched, seg)) {
            const XBwdUnit u = x_bwd_unit<kKeys>(p, seg);
            int st = x_bwd_live<kKeys>(p, u, u.t0);
            if (st >= u.t1) continue;
            ok = wait(kKeys ? &ctl->xy_full : &ctl->xt_full, n_seg & 1) && wait_z(j);
            if (!ok) break;
            issued = true;
            issue_t1(j);
            ok = wait_w(j);
            if (!ok) break;
            issue_t2(j);
            for (bool first = true; st < u.t1; first = false, ++j) {
                st = x_bwd_live<kKeys>(p, u, st + 1);
                const bool more = st < u.t1;
                // (the accumulators of the segment before have been read by the epilogue)
                if (kKeys) {
                    ok = wait(&ctl->p_full, j & 1) && (!first || n_seg == 0 || wait(&ctl->acc_free, (n_seg - 1) & 1));
                    if (!ok) break;
                    issue_a(kColA2, kColT1, lo_wm + ((j % kXWStages) * kTileBytes >> 4), !first);
                    tc_commit_elect(smem_u32(&ctl->w_empty[j % kXWStages]), leader);
                    if (more) {
                        ok = wait_z(j + 1);
                        if (!ok) break;
                        issue_t1(j + 1);
                    }
                    ok = wait(&ctl->ds_full, j & 1);
                } else {
                    if (more) {
                        ok = wait_z(j + 1) && wait(&ctl->p_full, j & 1);
                        if (!ok) break;
                        issue_t1(j + 1);
                    }
                    ok = wait(&ctl->ds_full, j & 1) && (!first || n_seg == 0 || wait(&ctl->acc_free, (n_seg - 1) & 1));
                }
                if (!ok) break;
                issue_a(kColA1, kColT2, lo_zm + ((j % kXZStages) * kTileBytes >> 4), !first);
                tc_commit_elect(smem_u32(&ctl->z_empty[j % kXZStages]), leader);
                if (more) {
                    ok = wait_w(j + 1);
                    if (!ok) break;
                    issue_t2(j + 1);
                }
            }
            if (!ok) break;
            tc_commit_elect(smem_u32(&ctl->acc_done), leader);
            ++n_seg;
        }
        if (!ok && issued) {
            int none = 0;
            volatile int* no_abort = &none;
            tc_commit_elect(smem_u32(&ctl->teardown), leader);
            mbar_wait(smem_u32(&ctl->teardown), 0, no_abort, nullptr, 100000000ull, 0);
        }
    } else if (warp == kXBwdCleanWarp && clean) {
        // =============================== masked rows of K ==================================
        bool ok = true;
        int j = 0;
        while (ok && cursor.next(p.sched, seg)) {
            const XBwdUnit u = x_bwd_unit<kKeys>(p, seg);
            const unsigned long long* row = p.words + static_cast<long long>(u.b) * n_words;
            for (int t = u.t0; t < u.t1; ++t, ++j) {
                const int zs = j % kXZStages;
                const unsigned long long w0 = x_key_word(row, p.skv, 2 * t), w1 = x_key_word(row, p.skv, 2 * t + 1);
                ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&ctl->z_full[zs]), (j / kXZStages) & 1, s_abort, p.status, limit,
                                                       PA_DEV_TIMEOUT_PIPE));
                if (!ok) break;
                if ((w0 & w1) != ~0ull) {
                    x_zero_rows<kD>(smem_z + zs * kTileBytes, kHalfBytes, w0, lane);
                    x_zero_rows<kD>(smem_z + zs * kTileBytes + 64 * 128, kHalfBytes, w1, lane);
                    fence_proxy_async_shared();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->z_clean[zs]));
            }
        }
    } else if (warp < kXBwdSoftWarps) {
        // =============================== elementwise + epilogue ============================
        const int quarter = warp & 3, piece = warp >> 2;  // my lanes; my 32 columns
        const int row_in_tile = quarter * 32 + lane;
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t t1 = tmem + lane_base + kColT1 + piece * 32, t2 = tmem + lane_base + kColT2 + piece * 32;
        // (dS and P of my 32 columns are packed into the first 16 of them: no other warp reads or writes there)
        const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);
        // (a vote: it brings the lanes together again, and a wait that gives up in some of them must not split the warp)
        auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
            return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, s_abort, p.status, limit, PA_DEV_TIMEOUT_PIPE));
        };
        auto arrive = [&](uint64_t* bar) {
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(bar));
        };
        // Query pass: brings a segment's X and Y from shared memory to TMEM once its predecessor's products
        // are done: D / 8 16-byte chunks per row, four of them per warp. Then adds up do * out of the rows, each warp
        // for 8 of them, with whole rows per load (from registers, where a thread has a quarter of a row of do, the
        // loads of out take 32 lines each and the pass 35 us longer) and in the order of xattn_stat_kernel, so
        // that dk and dv do not depend on who adds up.
        int n_copied = 0;
        auto copy_xy = [&](const XBwdUnit& w) -> bool {
            constexpr int kLanes = kD / 8, kRows = 32 / kLanes, kTurns = 8 / kRows;
            const int chunk = lane % kLanes, dot_row = warp * 8 + lane / kLanes;  // in the tile; kRows on with every turn
            uint4 o[kTurns];
            const uint16_t* from = p.o + (w.b * p.o_s[0] + w.head * p.o_s[1]) + chunk * 8;
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                const int row = w.tile * kTileM + dot_row + i * kRows;
                o[i] = row < p.sq ? __ldg(reinterpret_cast<const uint4*>(from + row * p.o_s[2])) : make_uint4(0, 0, 0, 0);
            }
            const int lse_row = w.tile * kTileM + warp * 8 + (lane & 7);  // (behind the last query: as without any key)
            const float lse = lse_row < p.sq ? __ldg(p.lse + (static_cast<long long>(w.b) * p.hkv * p.group + w.head) * p.sq + lse_row) : -INFINITY;
            if (!wait(&ctl->xy_full, n_copied & 1)) return false;
            if (piece * 4 < kD / 8) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const uint8_t* src = smem + y * kTileBytes + (piece >> 1) * kHalfBytes + row_in_tile * 128;
                    uint32_t v[16];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 x = *reinterpret_cast<const uint4*>(src + (((((piece & 1) << 2) + i) ^ (row_in_tile & 7)) << 4));
                        v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
                    }
                    tmem_st16(tmem + lane_base + (y ? kColY : kColX) + piece * 16, v);
                }
                tc_wait_st();
            }
            tc_fence_before();
            arrive(&ctl->xt_full);
            const int shared_by = (p.kv_batch == 1 ? 0 : w.b) * p.hkv + p.by_group(w.head);  // (f16)
            float v_max = 0.f;
            unsigned largest = 0u;
            if constexpr (!kBF16) v_max = x_v_max(p, shared_by, lane);
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                const int r = dot_row + i * kRows;
                const uint4 y = *reinterpret_cast<const uint4*>(smem + kTileBytes + (chunk >> 3) * kHalfBytes + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
                const uint32_t xs[4] = {o[i].x, o[i].y, o[i].z, o[i].w}, ys[4] = {y.x, y.y, y.z, y.w};
                float dot = dot8<kBF16>(xs, ys);
#pragma unroll
                for (int k = 1; k < kLanes; k <<= 1) dot += __shfl_xor_sync(0xffffffffu, dot, k);
                if (chunk == 0) stat[kTileM + r] = dot;
                if constexpr (!kBF16) {
                    float sum = abs8<kBF16>(ys);
#pragma unroll
                    for (int k = 1; k < kLanes; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
                    if (chunk == 0) stat[2 * kTileM + r] = static_cast<float>(x_slope_exp(sum * v_max));
                    // (rows without any key: as in xattn_stat_kernel)
                    const float its_lse = __shfl_sync(0xffffffffu, lse, lane / kLanes + i * kRows);
                    if (sum < INFINITY && its_lse != -INFINITY) largest = max(largest, __float_as_uint(sum));
                }
            }
            if constexpr (!kBF16) {
                largest = __reduce_max_sync(0xffffffffu, largest);
                if (lane == 0) atomicMax(p.do_max + shared_by, largest);
            }
            if (lane < 8) stat[warp * 8 + lane] = lse;
            arrive(&ctl->stat_full);
            ++n_copied;
            return true;
        };
        // Tells the producer that the owned tiles' memory may be loaded again (the stores staged there have been read).
        bool owe_release = false;
        auto release_xy = [&]() {
            if (owe_release && lane == 0) {
                tma_store_wait_read();
                mbar_arrive(smem_u32(&ctl->xy_empty));
            }
            owe_release = false;
        };
        bool ok = true;
        int j = 0, n_seg = 0;
        float2 neg = make_float2(0.f, 0.f), dl = make_float2(0.f, 0.f);
        // f16: query pass, 2^-e of my row, which A1 is to be multiplied by; key pass, 2^(e - kXShiftP), which makes dS of
        // P (dP - delta) with P as it is handed over
        float shift = 1.f;
        while (ok && cursor.next(p.sched, seg)) {
            const XBwdUnit u = x_bwd_unit<kKeys>(p, seg);
            int st = x_bwd_live<kKeys>(p, u, u.t0);
            const bool any = st < u.t1;
            if (!kKeys && any && n_seg == 0) {
                ok = copy_xy(u);
                if (!ok) break;
                owe_release = true;
            }
            const int row = u.tile * kTileM + row_in_tile;  // my query (query pass) or key (key pass)
            if (!kKeys && any) {
                ok = wait(&ctl->stat_full, n_seg & 1);
                if (!ok) break;
                const float lse = stat[row_in_tile], dot = stat[kTileM + row_in_tile];
                const bool none = lse == -INFINITY;
                float n1 = none ? -INFINITY : __fmul_rn(lse, -1.4426950408889634f);
                const float d1 = none ? 0.f : -dot;
                neg = make_float2(n1, n1);
                dl = make_float2(d1, d1);
                if constexpr (!kBF16) {  // (here P is in dS alone)
                    const float e = stat[2 * kTileM + row_in_tile];
                    neg = make_float2(n1 + e, n1 + e);
                    shift = x_pow2(-static_cast<int>(e));
                    n1 = __fadd_rn(n1, kXShiftP);
                }
                if (piece == 0 && u.t0 == 0) {  // for the key pass (a unit has one segment with its first step)
                    float* dst = p.stats + ((static_cast<long long>(u.b) * p.hkv * p.group + u.head) * p.mt + u.tile) * (2 * kTileN) + row_in_tile;
                    dst[0] = n1;
                    dst[kTileN] = d1;
                }
            }
            if constexpr (!kBF16 && kKeys) {
                const int unit = u.b * p.hkv + u.head;
                const int e = x_slope_exp(__uint_as_float(__ldcg(p.do_max + unit)) * x_v_max(p, unit, lane));
                shift = x_pow2(e - kXShiftP);
            }
            const bool whole = p.words == nullptr && (!kKeys || (u.tile + 1) * kTileM <= p.skv);  // every owned key takes part
            while (st < u.t1) {
                uint32_t live = 0xffffffffu;  // query pass: my columns' keys; key pass: all or nothing
                if (whole && (kKeys || (st + 1) * kTileN <= p.skv)) {
                } else if (!kKeys) {
                    live = static_cast<uint32_t>(x_key_word(p.words != nullptr ? p.words + static_cast<long long>(u.b) * n_words : nullptr,
                                                            p.skv, 2 * st + (piece >> 1)) >> ((piece & 1) * 32));
                } else if (p.words != nullptr) {
                    const int b = x_bwd_step<kKeys>(p, u, st).b;
                    if (row >= p.skv || ((__ldg(p.words + static_cast<long long>(b) * n_words + (row >> 6)) >> (row & 63)) & 1ull) == 0) live = 0u;
                } else if (row >= p.skv) {
                    live = 0u;
                }
                // (code of its own for steps without a mask: with tests inside the loops the query pass took 525 instead of
                // 484 us at 32760 x 512 x 40 heads)
                const bool plain = __all_sync(0xffffffffu, live == 0xffffffffu);
                // (key pass: the step's statistics come with W)
                const float4* cl = reinterpret_cast<const float4*>(stat + (j % kXWStages) * 2 * kTileN + piece * 32);
                if (kKeys) ok = wait(&ctl->w_full[j % kXWStages], (j / kXWStages) & 1) && ok;
                ok = wait(&ctl->t1_full, j & 1) && ok;
                tc_fence_after();
                uint32_t a[32];
                tmem_ld32(t1, a);
                tc_wait_ld();
                tmem_ld_fence(a);
                if (!kKeys) {
                    tc_fence_before();
                    arrive(&ctl->p_full);
                }
                auto weights = [&](auto all) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float2 ng[2] = {neg, neg};
                        if (kKeys) {
                            const float4 l4 = cl[i >> 2];
                            ng[0] = make_float2(l4.x, l4.y);
                            ng[1] = make_float2(l4.z, l4.w);
                        }
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const int c = i + 2 * y;
                            const float2 x = __ffma2_rn(make_float2(__uint_as_float(a[c]), __uint_as_float(a[c + 1])), sl2, ng[y]);
                            float e0 = ex2_approx(x.x), e1 = ex2_approx(x.y);
                            if (!decltype(all)::value && !(kKeys && plain)) {
                                if (((live >> c) & 1u) == 0) e0 = 0.f;
                                if (((live >> (c + 1)) & 1u) == 0) e1 = 0.f;
                            }
                            a[c] = __float_as_uint(e0);
                            a[c + 1] = __float_as_uint(e1);
                        }
                    }
                };
                if (!kKeys && plain) weights(std::true_type());
                else weights(std::false_type());
                if (kKeys) {
                    uint32_t pp[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        pp[i] = kBF16 ? pack_bf16x2(__uint_as_float(a[2 * i]), __uint_as_float(a[2 * i + 1]))
                                      : pack_f16x2(__uint_as_float(a[2 * i]), __uint_as_float(a[2 * i + 1]));
                    tmem_st16(t1, pp);
                    tc_wait_st();
                    tc_fence_before();
                    arrive(&ctl->p_full);
                }
                ok = wait(&ctl->t2_full, j & 1) && ok;
                tc_fence_after();
                uint32_t d[32], ds[16];
                tmem_ld32(t2, d);
                tc_wait_ld();
                tmem_ld_fence(d);
                auto slopes = [&](auto all) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float2 dt[2] = {dl, dl};
                        if (kKeys) {
                            const float4 d4 = cl[(i >> 2) + kTileN / 4];
                            dt[0] = make_float2(d4.x, d4.y);
                            dt[1] = make_float2(d4.z, d4.w);
                        }
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const int c = i + 2 * y;
                            float2 w = make_float2(__uint_as_float(a[c]), __uint_as_float(a[c + 1]));
                            if constexpr (!kBF16 && kKeys) w = __fmul2_rn(w, make_float2(shift, shift));
                            float2 s = __fmul2_rn(w, __fadd2_rn(make_float2(__uint_as_float(d[c]), __uint_as_float(d[c + 1])), dt[y]));
                            if (!decltype(all)::value && !(kKeys && plain)) {  // (T2 of a masked key may be anything)
                                if (((live >> c) & 1u) == 0) s.x = 0.f;
                                if (((live >> (c + 1)) & 1u) == 0) s.y = 0.f;
                            }
                            ds[c >> 1] = kBF16 ? pack_bf16x2(s.x, s.y) : pack_f16x2(s.x, s.y);
                        }
                    }
                };
                if (!kKeys && plain) slopes(std::true_type());
                else slopes(std::false_type());
                tmem_st16(t2, ds);
                tc_wait_st();
                tc_fence_before();
                arrive(&ctl->ds_full);
                if (kKeys && lane == 0) mbar_arrive(smem_u32(&ctl->w_empty[j % kXWStages]));
                if (!ok) break;
                if (!kKeys) release_xy();  // (behind the first step: the stores have long been read by then)
                ++j;
                st = x_bwd_live<kKeys>(p, u, st + 1);
            }
            if (!ok) break;
            bool copied = false;
            if (any) {
                // The last T2 is there, so X and Y in TMEM are free: the next segment's first products follow this
                // one's last in the tensor core's queue and run during this one's epilogue.
                XBwdUnit next;
                if (!kKeys && x_bwd_more<kKeys>(p, cursor, next)) {
                    ok = copy_xy(next);
                    if (!ok) break;
                    copied = true;
                }
                ok = wait(&ctl->acc_done, n_seg & 1);
                // (the epilogue reuses the memory that X and Y were copied from: by all warps, first)
                if (copied) ok = wait(&ctl->xt_full, (n_copied - 1) & 1) && ok;
                if (!ok) break;
                tc_fence_after();
                ++n_seg;
            }
            // Each warp writes blocks of 32 rows x 32 columns: the query pass's one of dq, the key pass's two of dk and
            // dv; staged where the owned tiles (query pass: X alone) were, which are no longer needed.
            constexpr int kBlocks = (kKeys ? 2 : 1) * kD / 32;  // of 32 columns
            static_assert(kXBwdSoftWarps * ((kBlocks + 3) / 4) * kXStageBytes <= (kKeys ? 2 : 1) * kTileBytes, "the staging fits");
            const int row_w = u.tile * kTileM + quarter * 32, rows = kKeys ? p.skv : p.sq;
            // (2^-e from 2^(e - kXShiftP): a difference of exponents)
            const float undo = kBF16 ? 1.0f : kKeys ? __uint_as_float((static_cast<unsigned>(254 - kXShiftP) << 23) - __float_as_uint(shift)) : shift;
            const float undo_p = kBF16 ? 1.0f : x_pow2(-kXShiftP);
#pragma unroll
            for (int blk = piece; blk < kBlocks; blk += 4) {
                const int which = blk / (kD / 32), col = blk % (kD / 32) * 32;
                if (!any && seg.slot < 0) {
                    // nothing to add up: zeros, stored directly (the memory may hold the next owned tiles)
                    if (row < rows) {
                        uint4* dst = reinterpret_cast<uint4*>(p.g[which] + (u.b * p.g_sb[which] + u.head * p.g_sh[which] + row * p.g_ss[which]) + col);
#pragma unroll
                        for (int x = 0; x < 4; ++x) dst[x] = make_uint4(0, 0, 0, 0);
                    }
                    continue;
                }
                uint32_t o[32];
                tmem_ld32(tmem + lane_base + (which ? kColA2 : kColA1) + col, o);
                tc_wait_ld();
                tmem_ld_fence(o);
                if (!any) {
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = 0u;
                }
                if (seg.slot < 0) {
                    uint8_t* stage = smem + (warp * (kKeys ? 2 : 1) + blk / 4) * kXStageBytes;
                    x_stage32<kBF16>(stage, lane, o, which ? undo_p : p.scale * undo);
                    fence_proxy_async_shared();
                    __syncwarp();
                    if (lane == 0 && row_w < rows)
                        tma_store_5d(which ? &tm_g1 : &tm_g0, smem_u32(stage), col, row_w, u.head, u.b, 0);
                } else {
                    if constexpr (!kBF16) {  // (the joining kernel adds up what the values are)
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * (which ? undo_p : undo));
                    }
                    float4* part = reinterpret_cast<float4*>(p.part) +
                                   ((static_cast<long long>(seg.slot) * 2 + which) * (kD / 4) + col / 4) * kTileM + row_in_tile;
#pragma unroll
                    for (int v4 = 0; v4 < 8; ++v4)
                        __stcg(part + v4 * kTileM,
                               make_float4(__uint_as_float(o[4 * v4]), __uint_as_float(o[4 * v4 + 1]),
                                           __uint_as_float(o[4 * v4 + 2]), __uint_as_float(o[4 * v4 + 3])));
                }
            }
            if (any) {
                tc_fence_before();
                arrive(&ctl->acc_free);
                // The owned tiles' memory may be loaded again: key pass, with the next ones; query pass, with those
                // behind the ones already copied.
                owe_release = kKeys || copied;
                if (kKeys) release_xy();
            }
        }
        if (lane == 0) tma_store_wait();
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) x_report(p.status_host, ctl->abort);
    if (warp == kXBwdMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// Adds the partial results of units that several CTAs worked on, in range order: one block per
// cut unit, 8 columns and accumulator, one thread per row.
template <bool kBF16, int kD, bool kKeys>
__global__ void __launch_bounds__(128)
xattn_bwd_join_kernel(const __grid_constant__ XBwdParams p, const __grid_constant__ XCutList cuts) {
    const XCut cut = cuts.cut[blockIdx.x];
    const int unit = cut.unit, cols0 = blockIdx.y * 8, which = blockIdx.z, r = threadIdx.x;
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    x_for_parts(p.sched, cut, [&](int slot) {
            const float4* src = reinterpret_cast<const float4*>(p.part) +
                                ((static_cast<long long>(slot) * 2 + which) * (kD / 4) + cols0 / 4) * kTileM + r;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const float4 x = __ldcg(src + v * kTileM);
                acc[4 * v] += x.x;
                acc[4 * v + 1] += x.y;
                acc[4 * v + 2] += x.z;
                acc[4 * v + 3] += x.w;
            }
        });
    XSeg g;
    g.unit = unit;
    g.t0 = g.t1 = 0;
    const XBwdUnit u = x_bwd_unit<kKeys>(p, g);
    const int row = u.tile * kTileM + r;
    if (row >= (kKeys ? p.skv : p.sq)) return;
    const float factor = which ? 1.0f : p.scale;
    uint16_t* grow = p.g[which] + (u.b * p.g_sb[which] + u.head * p.g_sh[which] + row * p.g_ss[which]) + cols0;
    uint32_t q[4];
#pragma unroll
    for (int x = 0; x < 4; ++x)
        q[x] = kBF16 ? pack_bf16x2(acc[2 * x] * factor, acc[2 * x + 1] * factor) : pack_f16x2(acc[2 * x] * factor, acc[2 * x + 1] * factor);
    *reinterpret_cast<uint4*>(grow) = make_uint4(q[0], q[1], q[2], q[3]);
}

// f16: v_max[kv batch][kv head][part] = the largest finite |v| of the keys of the part that take part in any batch entry
// that shares them, and a cleared do_max. One block per (kv batch, kv head) and part, 16 bytes per lane, HBM-bound:
// v is read once more. 2.2 us for 2 x 77 keys x 16 heads of 64, 4.9 us for 512 keys x 40 heads of 128; where v is the largest
// tensor it shows (256 queries x 32760 keys x 24 heads: the backward call takes 516 instead of 474 us).
struct XBoundParams {
    const uint16_t* v;
    long long v_s[3];
    const unsigned long long* words;
    int batch, kv_batch, hkv, skv;
    int keys;  // of a part
    unsigned *v_max, *do_max;
};
constexpr int kXBoundThreads = 256;
template <int kD>
__global__ void __launch_bounds__(kXBoundThreads)
xattn_bound_kernel(const __grid_constant__ XBoundParams p) {
    constexpr int kLanes = kD / 8;
    __shared__ unsigned of_warp[kXBoundThreads / 32];
    const int b = blockIdx.x / p.hkv, h = blockIdx.x - b * p.hkv, n_words = (p.skv + 63) >> 6;
    const int first = blockIdx.y * p.keys, end = min(first + p.keys, p.skv);
    const int b0 = p.kv_batch == 1 ? 0 : b, b1 = p.kv_batch == 1 ? p.batch : b + 1;
    const uint16_t* from = p.v + b * p.v_s[0] + h * p.v_s[1] + threadIdx.x % kLanes * 8;
    float m = 0.f;
#pragma unroll 4
    for (int key = first + threadIdx.x / kLanes; key < end; key += kXBoundThreads / kLanes) {
        bool live = p.words == nullptr;
        for (int bb = b0; bb < b1 && !live; ++bb)
            live = ((__ldg(p.words + static_cast<long long>(bb) * n_words + (key >> 6)) >> (key & 63)) & 1ull) != 0;
        const uint4 x = live ? __ldg(reinterpret_cast<const uint4*>(from + key * p.v_s[2])) : make_uint4(0, 0, 0, 0);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lo = fabsf(lo16<false>(xs[i])), hi = fabsf(hi16<false>(xs[i]));
            m = fmaxf(m, fmaxf(lo < INFINITY ? lo : 0.f, hi < INFINITY ? hi : 0.f));
        }
    }
    const unsigned w = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
    if (threadIdx.x % 32 == 0) of_warp[threadIdx.x / 32] = w;
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned all = of_warp[0];
#pragma unroll
        for (int i = 1; i < kXBoundThreads / 32; ++i) all = max(all, of_warp[i]);
        p.v_max[static_cast<long long>(blockIdx.x) * kXBoundParts + blockIdx.y] = all;
        if (blockIdx.y == 0) p.do_max[blockIdx.x] = 0u;
    }
}

// stats[b][h][tile][0 / 1][128] = -lse * log2 e (in f16, + the exponent of P) and -sum_d do * out of the query rows; (-inf, 0) for rows without
// any key and behind the last one; for calls without a query pass. HBM-bound: one pass over do and out, 16 bytes
// per lane.
struct XStatParams {
    const uint16_t *o, *g;  // out, do
    long long o_s[3], g_s[3];
    const float* lse;  // [B][Hq][Sq]
    float* stats;      // [B][Hq][padded / 128][2][128]
    unsigned* do_max;  // f16: XBwdParams::do_max
    int batch, heads, sq, padded;
    int kv_batch, hkv;
    XDiv by_group;
};
constexpr int kXStatThreads = 256;
// f16: each CTA finds the largest rows of its key heads in shared memory first (a look at the global word for every
// row made the kernel's 128 us 301 us at 32760 x 512 x 40 heads; so it is 149 us), if there are no more of them than this.
constexpr int kXStatUnits = 1024;
template <bool kBF16, int kD>
__global__ void __launch_bounds__(kXStatThreads)
xattn_stat_kernel(const __grid_constant__ XStatParams p) {
    constexpr int kLanes = kD / 8;
    const int at = (threadIdx.x % kLanes) * 8;
    constexpr int kAtOnce = 4;  // vectors per lane in flight
    constexpr unsigned kGroups = kXStatThreads / kLanes;
    const unsigned n = static_cast<unsigned>(p.batch) * p.heads * p.padded;  // (the host has checked the range)
    __shared__ unsigned most[kBF16 ? 1 : kXStatUnits];
    const int units = p.kv_batch * p.hkv;
    const bool here = units <= kXStatUnits;
    if constexpr (!kBF16) {
        for (int i = threadIdx.x; i < units && here; i += kXStatThreads) most[i] = 0u;
        __syncthreads();
    }
    // (heads innermost: neighbouring lanes read neighbouring heads of [B, S, H, D] memory. The trip count
    // is the same for all lanes of a warp - the shuffles need them all.)
    for (unsigned base = blockIdx.x * (kGroups * kAtOnce); base < n; base += gridDim.x * (kGroups * kAtOnce)) {
        uint4 x[kAtOnce], y[kAtOnce];
        float l[kAtOnce];
        unsigned to[kAtOnce];
        int unit[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const unsigned idx = base + u * kGroups + threadIdx.x / kLanes;
            const unsigned t = idx / static_cast<unsigned>(p.heads);
            const int h = static_cast<int>(idx - t * p.heads);
            const int b = static_cast<int>(t / static_cast<unsigned>(p.padded));
            const int s = static_cast<int>(t) - b * p.padded;
            x[u] = y[u] = make_uint4(0, 0, 0, 0);
            l[u] = -INFINITY;  // (behind the last query, as without any key)
            unit[u] = kBF16 ? 0 : (p.kv_batch == 1 ? 0 : b) * p.hkv + p.by_group(h);
            to[u] = idx < n ? (static_cast<unsigned>(b) * p.heads + h) * p.padded + s : ~0u;
            if (idx < n && s < p.sq) {
                x[u] = __ldg(reinterpret_cast<const uint4*>(p.o + (b * p.o_s[0] + h * p.o_s[1] + s * p.o_s[2]) + at));
                y[u] = __ldg(reinterpret_cast<const uint4*>(p.g + (b * p.g_s[0] + h * p.g_s[1] + s * p.g_s[2]) + at));
                l[u] = __ldg(p.lse + (static_cast<long long>(b) * p.heads + h) * p.sq + s);
            }
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const uint32_t xs[4] = {x[u].x, x[u].y, x[u].z, x[u].w}, ys[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
            float dot = dot8<kBF16>(xs, ys);
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            float sum = 0.f;
            if constexpr (!kBF16) {
                sum = abs8<kBF16>(ys);
#pragma unroll
                for (int o = 1; o < kLanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            }
            if (at == 0 && to[u] != ~0u) {
                const bool none = l[u] == -INFINITY;
                float* dst = p.stats + static_cast<long long>(to[u] / kTileN) * (2 * kTileN) + to[u] % kTileN;
                // (two roundings, as in the query pass)
                const float n1 = __fmul_rn(l[u], -1.4426950408889634f);
                dst[0] = none ? -INFINITY : kBF16 ? n1 : __fadd_rn(n1, kXShiftP);
                dst[kTileN] = none ? 0.f : -dot;
                if constexpr (!kBF16) {
                    if (!none && sum < INFINITY) {
                        if (here) atomicMax(most + unit[u], __float_as_uint(sum));
                        else if (__float_as_uint(sum) > __ldcg(p.do_max + unit[u])) atomicMax(p.do_max + unit[u], __float_as_uint(sum));
                    }
                }
            }
        }
    }
    if constexpr (!kBF16) {
        __syncthreads();
        for (int i = threadIdx.x; i < units && here; i += kXStatThreads)
            if (most[i] != 0u) atomicMax(p.do_max + i, most[i]);
    }
}

}  // namespace pa
