// Cross attention forward for B200: out = softmax(scale q k^T + mask) v and its log-sum-exp,
// tcgen05 with TMEM accumulators, TMA loads, persistent CTAs.
//
// Why not the long-sequence kernel of attn_fwd_sm100.cuh: an encoder's states are short. 512 keys
// are four key tiles, 7 us of work, and a CTA of that kernel spends 16 us around its loop (setup,
// TMEM allocation, the first loads, the epilogue), none of it overlapped. Here one CTA per SM
// stays resident and walks many units, and the roles run ahead of each other across units: while
// the softmax warps write a unit's output, the tensor core already computes the next unit's first
// Q K^T and the loads behind it are in flight.
//
// A unit is two row tiles of 128 queries that share a key / value head: tile i of (batch, kv head)
// is query head i / mt, rows (i % mt) * 128, mt = ceil(Sq / 128) - so with short queries two heads
// of a group share one pass over the keys. The two tiles take turns: while one is in its softmax the
// tensor core runs the other's P V and next Q K^T.
//
// Two threads share a row, 64 key columns each (16 softmax warps). That halves the softmax's latency,
// which is what lets Q K^T run on whole tiles: the long kernel's one thread per row is too slow for that
// and splits Q K^T into N = 64 halves, which cost 66 cycles of shared-memory operand fetch each instead of
// 32 (3136 cycles of products per key tile and unit instead of 2048). The threads of a row meet once per
// key tile, to agree on its maximum; O is rescaled lazily, when a row outgrows the reference its weights
// are relative to by more than 2^8.
//
// Warps: 0-15 softmax and epilogue (tile w / 8, columns half (w / 4) % 2, TMEM lane quarter w % 4), 16 MMA
// issuer, 17 TMA producer, 18 clears masked rows of V (only with a mask). TMEM columns: S0 S1 [0,256),
// O0 O1 [256, 256 + 2 D); P overwrites S.
//
// Bounds: bytes q, k, v read + out written once at HBM rate, or 4 Sq Skv D flops per head at the
// tensor rate. A unit re-reads its head's K and V from L2.
#pragma once
#include "xattn_sm100.cuh"

namespace pa {

constexpr int kXFwdSoftWarps = 16;
constexpr int kXFwdMmaWarp = 16, kXFwdTmaWarp = 17, kXFwdCleanWarp = 18;
constexpr int kXFwdThreads = 640;

struct XFwdParams {
    int kv_batch, hkv, group, sq, skv, mt;
    float scale, scale_log2;
    uint16_t* out;  // (the joining kernel's; the main kernel stores through its tensor map)
    long long o_sb, o_sh, o_ss;
    float* lse;  // [B][Hq][Sq] or NULL
    const unsigned long long* words;  // key mask, or NULL
    const int* extent;
    XSched sched;
    XDiv by_pairs, by_hkv, by_mt;  // pairs: of row tiles of a (batch entry, kv head)
    float* part_o;    // [slot][D / 4][256 rows][4]
    float2* part_ml;  // [slot][256 rows] (reference, row sum)
    int* status;
    int* status_host;
    unsigned long long wait_ns;
};

struct XFwdCtl {
    uint64_t q_full, q_empty;
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], v_clean[2];
    uint64_t s_full[2];     // Q K^T of a row tile is in TMEM
    uint64_t p_full[2];     // P of a row tile is in TMEM and its O is rescaled (one arrival per warp)
    uint64_t o_done[2];     // P V of a row tile (and every product before it) is done
    uint64_t teardown;
    uint32_t tmem_base;
    int abort;
};
// Q, K and V ring; output staging, one buffer for each softmax warp; what the two threads of a row exchange; control
// block. (The dynamic shared memory is declared with the alignment of the swizzle; there is no room for slack.)
constexpr int kXFwdSmemBytes = 6 * kTileBytes + kXFwdSoftWarps * kXStageBytes + kXFwdSoftWarps * 32 * 4 + 512;
static_assert(sizeof(XFwdCtl) <= 512, "control block too large");
static_assert(kXFwdSmemBytes <= 232448, "shared memory");

// What a segment of work means: which rows, which keys.
struct XFwdUnit {
    int b, hk, tile0;  // first of the two row tiles of (b, hk)
    int lo, hi;        // key tiles
};
__device__ __forceinline__ XFwdUnit x_fwd_unit(const XFwdParams& p, const XSeg& g) {
    XFwdUnit u;
    const int x = p.by_pairs(g.unit);
    u.tile0 = 2 * (g.unit - x * static_cast<int>(p.by_pairs.d));
    u.b = p.by_hkv(x);
    u.hk = x - u.b * p.hkv;
    u.lo = g.t0;
    u.hi = g.t1;
    if (p.extent != nullptr) {
        const int n = (__ldg(p.extent + u.b) + kTileN - 1) / kTileN;
        u.hi = min(u.hi, n);
        u.lo = min(u.lo, u.hi);
    }
    return u;
}

template <bool kBF16, int kD>
__global__ void __launch_bounds__(kXFwdThreads, 1)
xattn_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                 const __grid_constant__ XFwdParams p) {
    constexpr int kAtoms = kD / 64;
    constexpr int kOperandBytes = kAtoms * kHalfBytes;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sQ = smem_u32(smem);
    const uint32_t sK = sQ + 2 * kTileBytes;
    const uint32_t sV = sK + 2 * kTileBytes;
    float* exchange = reinterpret_cast<float*>(smem + 6 * kTileBytes + kXFwdSoftWarps * kXStageBytes);  // [warp][32]
    XFwdCtl* ctl = reinterpret_cast<XFwdCtl*>(exchange + kXFwdSoftWarps * 32);
    volatile int* s_abort = &ctl->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        int st = p.status != nullptr ? *reinterpret_cast<volatile int*>(p.status) : 0;
        if ((sQ & 1023u) != 0) {  // (never seen; the swizzled tiles would not be where the descriptors say)
            st = PA_DEV_TIMEOUT_PIPE;
            if (p.status != nullptr) atomicCAS(p.status, 0, st);
        }
        x_report(p.status_host, st);  // (a launch that does nothing because of an earlier one's wait says so, too)
        ctl->abort = st;
    }
    __syncthreads();
    if (ctl->abort != 0) return;
    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&ctl->q_full), 1);
        mbar_init(smem_u32(&ctl->q_empty), 1);
        for (int s = 0; s < 2; ++s) {
            mbar_init(smem_u32(&ctl->k_full[s]), 1);
            mbar_init(smem_u32(&ctl->k_empty[s]), 1);
            mbar_init(smem_u32(&ctl->v_full[s]), 1);
            mbar_init(smem_u32(&ctl->v_empty[s]), 1);
            mbar_init(smem_u32(&ctl->v_clean[s]), 1);
            mbar_init(smem_u32(&ctl->s_full[s]), 1);
            mbar_init(smem_u32(&ctl->p_full[s]), 8);
            mbar_init(smem_u32(&ctl->o_done[s]), 1);
        }
        mbar_init(smem_u32(&ctl->teardown), 1);
        mbar_init_fence();
    }
    if (warp == kXFwdMmaWarp) {
        tmem_alloc(smem_u32(&ctl->tmem_base), kTmemCols);
        tmem_relinquish();
    }
    if (warp == kXFwdTmaWarp && lane == 0) {
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        tma_prefetch_desc(&tm_o);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;
    const uint64_t limit = p.wait_ns;
    const int n_words = (p.skv + 63) >> 6;

    XCursor cursor(p.sched);
    XSeg seg;
    if (warp == kXFwdTmaWarp) {
        // =============================== TMA producer ======================================
        if (lane == 0) {
            bool ok = true;
            int j = 0, u = 0;  // key tiles and units loaded so far
            while (ok && cursor.next(p.sched, seg)) {
                const XFwdUnit w = x_fwd_unit(p, seg);
                if (w.lo >= w.hi) continue;
                if (u > 0) ok = mbar_wait(smem_u32(&ctl->q_empty), (u - 1) & 1, s_abort, p.status, limit, PA_DEV_TIMEOUT_PIPE);
                if (!ok) break;
                const uint32_t bq = smem_u32(&ctl->q_full);
                mbar_expect_tx(bq, 2 * kOperandBytes);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    // (a second tile that does not exist is loaded from behind the last row: zeros)
                    const int i = w.tile0 + t, g = p.by_mt(i);
                    const bool real = g < p.group;
                    const int row = real ? (i - g * p.mt) * kTileM : p.mt * kTileM;
#pragma unroll
                    for (int h = 0; h < kAtoms; ++h)
                        tma_load_5d(sQ + t * kTileBytes + h * kHalfBytes, &tm_q, bq, h * 64, row,
                                    w.hk * p.group + (real ? g : 0), w.b, 0);
                }
                const int bk_ = p.kv_batch == 1 ? 0 : w.b;
                for (int t = w.lo; t < w.hi && ok; ++t, ++j) {
                    const int st = j & 1;
                    const uint32_t ph = (j >> 1) & 1;
                    const uint32_t bk = smem_u32(&ctl->k_full[st]), bv = smem_u32(&ctl->v_full[st]);
                    if (j >= 2) ok = mbar_wait(smem_u32(&ctl->k_empty[st]), ph ^ 1, s_abort, p.status, limit, PA_DEV_TIMEOUT_PIPE);
                    if (!ok) break;
                    mbar_expect_tx(bk, kOperandBytes);
#pragma unroll
                    for (int h = 0; h < kAtoms; ++h)
                        tma_load_5d(sK + st * kTileBytes + h * kHalfBytes, &tm_k, bk, h * 64, t * kTileN, w.hk, bk_, 0);
                    if (j >= 2) ok = mbar_wait(smem_u32(&ctl->v_empty[st]), ph ^ 1, s_abort, p.status, limit, PA_DEV_TIMEOUT_PIPE);
                    if (!ok) break;
                    mbar_expect_tx(bv, kOperandBytes);
#pragma unroll
                    for (int h = 0; h < kAtoms; ++h)
                        tma_load_5d(sV + st * kTileBytes + h * kHalfBytes, &tm_v, bv, h * 64, t * kTileN, w.hk, bk_, 0);
                }
                ++u;
            }
            if (*s_abort != 0) {
                // Leave only once copies already issued have landed (bounded): every barrier's phase
                // that may still be open is given the time a copy can take.
                int none = 0;
                volatile int* no_abort = &none;
                if (u > 0 || j > 0) mbar_wait(smem_u32(&ctl->q_full), u > 0 ? (u - 1) & 1 : 0, no_abort, nullptr, 10000000ull, 0);
                mbar_wait(smem_u32(&ctl->q_full), u & 1, no_abort, nullptr, 10000000ull, 0);
                for (int jj = (j > 2 ? j - 2 : 0); jj <= j; ++jj) {
                    mbar_wait(smem_u32(&ctl->k_full[jj & 1]), (jj >> 1) & 1, no_abort, nullptr, 10000000ull, 0);
                    mbar_wait(smem_u32(&ctl->v_full[jj & 1]), (jj >> 1) & 1, no_abort, nullptr, 10000000ull, 0);
                }
            }
        }
    } else if (warp == kXFwdMmaWarp) {
        // =============================== MMA issuer ========================================
        constexpr uint32_t idesc_qk = make_idesc_f16(kBF16, false, kTileM, kTileN);
        constexpr uint32_t idesc_pv = make_idesc_f16(kBF16, true, kTileM, kD);
        const uint32_t leader = elect_one() ? 1u : 0u;
        const uint64_t dq0 = smem_desc_sw128(sQ, 16, 1024);
        const uint64_t dv0 = smem_desc_sw128(sV, kHalfBytes, 1024);
        const uint32_t hi_qk = static_cast<uint32_t>(dq0 >> 32), hi_v = static_cast<uint32_t>(dv0 >> 32);
        const uint32_t lo_q = static_cast<uint32_t>(dq0), lo_v = static_cast<uint32_t>(dv0);
        const uint32_t lo_k = static_cast<uint32_t>(smem_desc_sw128(sK, 16, 1024));
        auto issue_qk = [&](int t, int st) {
            const uint32_t a0 = lo_q + ((t * kTileBytes) >> 4), b0 = lo_k + ((st * kTileBytes) >> 4);
            const uint32_t d = tmem + kColS0 + t * kTileN;
#pragma unroll
            for (int ks = 0; ks < kD / 16; ++ks) {
                const uint32_t off = ((ks >> 2) * kHalfBytes + (ks & 3) * 32) >> 4;
                tc_mma_ss_elect(d, a0 + off, hi_qk, b0 + off, hi_qk, idesc_qk, ks > 0 ? 1u : 0u, leader);
            }
            tc_commit_elect(smem_u32(&ctl->s_full[t]), leader);
        };
        // 16 keys a k-step; their P is 8 packed columns (32 columns of S are packed into their first 16)
        auto issue_pv = [&](int t, int st, bool acc) {
            const uint32_t b0 = lo_v + ((st * kTileBytes) >> 4);
            const uint32_t a0 = tmem + kColS0 + t * kTileN;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
                tc_mma_ts_elect(tmem + kColO0 + t * kD, a0 + (ks >> 1) * 32 + (ks & 1) * 8, b0 + ((ks * 16 * 128) >> 4), hi_v,
                                idesc_pv, (acc || ks > 0) ? 1u : 0u, leader);
            tc_commit_elect(smem_u32(&ctl->o_done[t]), leader);
        };
        auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
            const bool r = mbar_wait(smem_u32(bar), parity, s_abort, p.status, limit, PA_DEV_TIMEOUT_PIPE);
            return __all_sync(0xffffffffu, r);
        };
        bool ok = true, issued = false;
        int j = 0, u = 0;
        while (ok && cursor.next(p.sched, seg)) {
            const XFwdUnit w = x_fwd_unit(p, seg);
            const int n = w.hi - w.lo;
            if (n <= 0) continue;
            ok = wait(&ctl->q_full, u & 1) && wait(&ctl->k_full[j & 1], (j >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
            issued = true;
            issue_qk(0, j & 1);
            issue_qk(1, j & 1);
            tc_commit_elect(smem_u32(&ctl->k_empty[j & 1]), leader);
            if (n == 1) tc_commit_elect(smem_u32(&ctl->q_empty), leader);
            for (int i = 0; i < n && ok; ++i, ++j) {
                const int st = j & 1, stn = (j + 1) & 1;
                const bool more = i + 1 < n;
                ok = wait(p.words != nullptr ? &ctl->v_clean[st] : &ctl->v_full[st], (j >> 1) & 1);
                if (ok && more) ok = wait(&ctl->k_full[stn], ((j + 1) >> 1) & 1);
                if (!ok) break;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    ok = wait(&ctl->p_full[t], j & 1);
                    if (!ok) break;
                    tc_fence_after();
                    issue_pv(t, st, i > 0);
                    if (t == 1) tc_commit_elect(smem_u32(&ctl->v_empty[st]), leader);
                    if (more) {
                        issue_qk(t, stn);
                        if (t == 1) {
                            tc_commit_elect(smem_u32(&ctl->k_empty[stn]), leader);
                            if (i + 2 == n) tc_commit_elect(smem_u32(&ctl->q_empty), leader);
                        }
                    }
                }
            }
            ++u;
        }
        if (!ok && issued) {
            // Nothing may still be running on the tensor core when TMEM is released.
            int none = 0;
            volatile int* no_abort = &none;
            tc_commit_elect(smem_u32(&ctl->teardown), leader);
            mbar_wait(smem_u32(&ctl->teardown), 0, no_abort, nullptr, 100000000ull, 0);
        }
    } else if (warp == kXFwdCleanWarp && p.words != nullptr) {
        // =============================== masked rows of V ==================================
        bool ok = true;
        int j = 0;
        while (ok && cursor.next(p.sched, seg)) {
            const XFwdUnit w = x_fwd_unit(p, seg);
            const unsigned long long* row = p.words + static_cast<long long>(w.b) * n_words;
            for (int t = w.lo; t < w.hi && ok; ++t, ++j) {
                const int st = j & 1;
                const unsigned long long w0 = x_key_word(row, p.skv, 2 * t);
                const unsigned long long w1 = x_key_word(row, p.skv, 2 * t + 1);
                ok = mbar_wait(smem_u32(&ctl->v_full[st]), (j >> 1) & 1, s_abort, p.status, limit, PA_DEV_TIMEOUT_PIPE);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if ((w0 & w1) != ~0ull) {
                    x_zero_rows<kD>(smem + 4 * kTileBytes + st * kTileBytes, kHalfBytes, w0, lane);
                    x_zero_rows<kD>(smem + 4 * kTileBytes + st * kTileBytes + 64 * 128, kHalfBytes, w1, lane);
                    fence_proxy_async_shared();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->v_clean[st]));
            }
        }
    } else if (warp < kXFwdSoftWarps) {
        // =============================== softmax + epilogue ================================
        // (Nobody leaves this loop early: the two warps of a row meet at named barriers, which both must reach the
        // same number of times. Once the abort word is set no wait blocks any more.)
        const int t = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3;
        const int row_in_tile = quarter * 32 + lane;
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t tS = tmem + lane_base + kColS0 + t * kTileN + half * 64;      // my 64 logits
        const uint32_t tO = tmem + lane_base + kColO0 + t * kD + half * (kD / 2);    // my half of the row's output
        float* mine = exchange + warp * 32 + lane;
        const float* other = exchange + (warp ^ 4) * 32 + lane;
        uint8_t* stage = smem + 6 * kTileBytes + warp * kXStageBytes;
        const float sl = p.scale_log2;
        auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + t * 4 + quarter) : "memory"); };
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, s_abort, p.status, limit, PA_DEV_TIMEOUT_PIPE));
        };
        int j = 0;
        while (cursor.next(p.sched, seg)) {
            const XFwdUnit w = x_fwd_unit(p, seg);
            const int n = w.hi - w.lo;
            const unsigned long long* mrow = p.words != nullptr ? p.words + static_cast<long long>(w.b) * n_words : nullptr;
            float m_ref = -INFINITY, l_sum = 0.f;
            for (int i = 0; i < n; ++i, ++j) {
                const unsigned long long word = x_key_word(mrow, p.skv, 2 * (w.lo + i) + half);
                const bool plain = word == ~0ull;  // (the same for the whole warp)
                wait(&ctl->s_full[t], j & 1);
                tc_fence_after();
                // Two passes over the logits, 32 at a time, the second in the opposite order: 96 registers do not
                // hold 64 of them, and reading TMEM again costs less than spilling.
                uint32_t sc[32];
                float mx[2] = {-INFINITY, -INFINITY};
                auto fetch = [&](int c) {
                    tmem_ld32(tS + c * 32, sc);
                    tc_wait_ld();
                    tmem_ld_fence(sc);
                    if (!plain) {
                        const uint32_t live = static_cast<uint32_t>(word >> (c * 32));
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (((live >> x) & 1u) == 0) sc[x] = __float_as_uint(-INFINITY);
                    }
                };
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    fetch(c);
#pragma unroll
                    for (int x = 0; x < 32; x += 4) {
                        mx[0] = fmax3(mx[0], __uint_as_float(sc[x]), __uint_as_float(sc[x + 1]));
                        mx[1] = fmax3(mx[1], __uint_as_float(sc[x + 2]), __uint_as_float(sc[x + 3]));
                    }
                }
                // The row's maximum. (The buffer needs no second copy: the next logits of this tile are there only
                // after both threads have handed over their P, that is, after both have read.)
                const float own = fmaxf(mx[0], mx[1]);
                *mine = own;
                meet();
                const float row_max = fmaxf(own, *other);
                const bool grow = (row_max - m_ref) * sl > kRescaleThreshold;  // (-inf - -inf: NaN, false)
                if (__any_sync(0xffffffffu, grow)) {  // (the same in both warps of the rows)
                    const float m_new = fmaxf(m_ref, row_max);
                    const float alpha = m_new == -INFINITY ? 1.0f : ex2_approx((m_ref - m_new) * sl);
                    m_ref = m_new;
                    l_sum *= alpha;
                    if (i > 0) {
                        wait(&ctl->o_done[t], (j - 1) & 1);
                        tc_fence_after();
#pragma unroll 1
                        for (int b = 0; b < kD / 64; ++b) {
                            uint32_t o[32];
                            tmem_ld32(tO + b * 32, o);
                            tc_wait_ld();
                            tmem_ld_fence(o);
#pragma unroll
                            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
                            tmem_st32(tO + b * 32, o);
                        }
                    }
                }
                const float neg = m_ref == -INFINITY ? 0.0f : -m_ref * sl;
                const float2 sl2 = make_float2(sl, sl), neg2 = make_float2(neg, neg);
                float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int c = 1; c >= 0; --c) {
                    if (c == 0) fetch(0);
                    uint32_t pk[16];
#pragma unroll
                    for (int x = 0; x < 32; x += 2) {
                        const float2 y = __ffma2_rn(make_float2(__uint_as_float(sc[x]), __uint_as_float(sc[x + 1])), sl2, neg2);
                        const float2 e = make_float2(ex2_approx(y.x), ex2_approx(y.y));
                        ls[(x >> 1) & 1] = __fadd2_rn(ls[(x >> 1) & 1], e);
                        pk[x >> 1] = kBF16 ? pack_bf16x2(e.x, e.y) : pack_f16x2(e.x, e.y);
                    }
                    tmem_st16(tS + c * 32, pk);
                }
                const float2 sum = __fadd2_rn(ls[0], ls[1]);
                l_sum += sum.x + sum.y;
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->p_full[t]));
            }
            // ---- the unit's output: my half of the row's columns -----------------------------------
            if (n > 0) wait(&ctl->o_done[t], (j - 1) & 1);
            tc_fence_after();
            *mine = l_sum;
            meet();
            l_sum += *other;
            const int tile = w.tile0 + t, g = p.by_mt(tile);
            const int row = (tile - g * p.mt) * kTileM + row_in_tile;
            const int head = w.hk * p.group + g;
            const bool none = n <= 0 || l_sum == 0.0f;  // no key at all: zeros, LSE -inf (a NaN sum stays one)
            const float inv = none ? 0.0f : 1.0f / l_sum;
            const int row_w = (tile - g * p.mt) * kTileM + quarter * 32;  // first of the warp's rows
#pragma unroll 1
            for (int b = 0; b < kD / 64; ++b) {
                uint32_t o[32];
                tmem_ld32(tO + b * 32, o);
                if (seg.slot < 0 && lane == 0) tma_store_wait_read();  // (the staging memory is free again)
                __syncwarp();
                tc_wait_ld();
                tmem_ld_fence(o);
                if (none) {
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = 0u;
                }
                const int col = half * (kD / 2) + b * 32;
                if (seg.slot < 0) {
                    x_stage32<kBF16>(stage, lane, o, inv);
                    fence_proxy_async_shared();
                    __syncwarp();
                    if (lane == 0 && g < p.group && row_w < p.sq) tma_store_5d(&tm_o, smem_u32(stage), col, row_w, head, w.b, 0);
                } else {  // this CTA's share of a unit: unnormalised O
                    float4* po = reinterpret_cast<float4*>(p.part_o) + static_cast<long long>(seg.slot) * (kD / 4) * 256 +
                                 (col / 4) * 256 + t * kTileM + row_in_tile;
#pragma unroll
                    for (int v4 = 0; v4 < 8; ++v4)
                        __stcg(po + v4 * 256, make_float4(__uint_as_float(o[4 * v4]), __uint_as_float(o[4 * v4 + 1]),
                                                          __uint_as_float(o[4 * v4 + 2]), __uint_as_float(o[4 * v4 + 3])));
                }
            }
            if (half == 0) {
                if (seg.slot >= 0)
                    __stcg(p.part_ml + static_cast<long long>(seg.slot) * 256 + t * kTileM + row_in_tile, make_float2(m_ref, l_sum));
                else if (p.lse != nullptr && g < p.group && row < p.sq)
                    p.lse[(static_cast<long long>(w.b) * p.hkv * p.group + head) * p.sq + row] =
                        none ? -INFINITY : m_ref * p.scale + logf(l_sum);
            }
            tc_fence_before();
            meet();  // (both have read the other's sum)
        }
        if (lane == 0) tma_store_wait();
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) x_report(p.status_host, ctl->abort);
    if (warp == kXFwdMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// Joins the partial results of units that several CTAs worked on (see XSched): one block per
// cut unit and 8 output columns, one thread per row.
//   out = sum_i 2^((m_i - m) sl) O_i / sum_i 2^((m_i - m) sl) l_i
template <bool kBF16, int kD>
__global__ void __launch_bounds__(256)
xattn_fwd_join_kernel(const __grid_constant__ XFwdParams p, const __grid_constant__ XCutList cuts) {
    const XCut cut = cuts.cut[blockIdx.x];
    const int unit = cut.unit, cols0 = blockIdx.y * 8, r256 = threadIdx.x;
    const float sl = p.scale_log2;
    float m = -INFINITY;
    x_for_parts(p.sched, cut, [&](int slot) { m = fmaxf(m, __ldcg(p.part_ml + static_cast<long long>(slot) * 256 + r256).x); });
    float acc[8], l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    x_for_parts(p.sched, cut, [&](int slot) {
        const float2 ml = __ldcg(p.part_ml + static_cast<long long>(slot) * 256 + r256);
        if (ml.y == 0.f) return;  // (a share that saw no key)
        const float wgt = exp2f((ml.x - m) * sl);
        l += ml.y * wgt;
        const float4* src = reinterpret_cast<const float4*>(p.part_o) +
                            (static_cast<long long>(slot) * (kD / 4) + cols0 / 4) * 256 + r256;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const float4 x = __ldcg(src + v * 256);
            acc[4 * v] = fmaf(x.x, wgt, acc[4 * v]);
            acc[4 * v + 1] = fmaf(x.y, wgt, acc[4 * v + 1]);
            acc[4 * v + 2] = fmaf(x.z, wgt, acc[4 * v + 2]);
            acc[4 * v + 3] = fmaf(x.w, wgt, acc[4 * v + 3]);
        }
    });
    XSeg g;
    g.unit = unit;
    g.t0 = g.t1 = 0;
    const XFwdUnit w = x_fwd_unit(p, g);
    const int tile = w.tile0 + (r256 >> 7), grp = p.by_mt(tile);
    const int row = (tile - grp * p.mt) * kTileM + (r256 & 127);
    if (grp >= p.group || row >= p.sq) return;
    const int head = w.hk * p.group + grp;
    const float inv = l != 0.f ? 1.f / l : 0.f;
    uint16_t* orow = p.out + (w.b * p.o_sb + head * p.o_sh + row * p.o_ss) + cols0;
    uint32_t q[4];
#pragma unroll
    for (int x = 0; x < 4; ++x)
        q[x] = kBF16 ? pack_bf16x2(acc[2 * x] * inv, acc[2 * x + 1] * inv) : pack_f16x2(acc[2 * x] * inv, acc[2 * x + 1] * inv);
    *reinterpret_cast<uint4*>(orow) = make_uint4(q[0], q[1], q[2], q[3]);
    if (blockIdx.y == 0 && p.lse != nullptr)
        p.lse[(static_cast<long long>(w.b) * p.hkv * p.group + head) * p.sq + row] =
            l != 0.f ? m * p.scale + logf(l) : -INFINITY;
}

}  // namespace pa
