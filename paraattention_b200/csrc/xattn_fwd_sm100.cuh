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
// of a group share one pass over the keys. Inside a unit the pipeline is that of the long kernel
// (half tiles in the key dimension, one-pass softmax in pieces of 32 columns, lazily rescaled O).
// Warps: 0-7 softmax (one thread per query row), 8 MMA issuer, 9 TMA producer, 10 clears masked
// rows of V (only with a mask). TMEM columns: S0 S1 [0,256), O0 O1 [256, 256 + 2 D).
//
// Bounds: bytes q, k, v read + out written once at HBM rate, or 4 Sq Skv D flops per head at the
// tensor rate. A unit re-reads its head's K and V from L2.
#pragma once
#include "xattn_sm100.cuh"

namespace pa {

struct XFwdParams {
    int batch, kv_batch, hkv, group, sq, skv, mt;
    float scale, scale_log2;
    uint16_t* out;  // (the joining kernel's; the main kernel stores through its tensor map)
    long long o_sb, o_sh, o_ss;
    float* lse;  // [B][Hq][Sq] or NULL
    const unsigned long long* words;  // key mask, or NULL
    const int* extent;
    XSched sched;
    float* part_o;    // [slot][D / 4][256 rows][4]
    float2* part_ml;  // [slot][256 rows] (reference, row sum)
    int* status;
    int* status_host;
    unsigned long long wait_ns;
};

struct XFwdCtl {
    uint64_t q_full, q_empty;
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], v_clean[2];
    uint64_t s_full[2][2];
    uint64_t p_full[2][kPieces];
    uint64_t o_done[2][kPieces];
    uint64_t teardown;
    uint32_t tmem_base;
    int abort;
};
// alignment slack; Q, K and V ring; output staging, two buffers for each softmax warp; control block
constexpr int kXFwdSmemBytes = 1024 + 6 * kTileBytes + 2 * kSoftmaxWarps * kXStageBytes + 512;
static_assert(kXFwdSmemBytes <= 232448, "shared memory");
static_assert(sizeof(XFwdCtl) <= 512, "control block too large");

// What a segment of work means: which rows, which keys.
struct XFwdUnit {
    int b, hk, tile0;  // first of the two row tiles of (b, hk)
    int lo, hi;        // key tiles
};
__device__ __forceinline__ XFwdUnit x_fwd_unit(const XFwdParams& p, const XSeg& g) {
    const int tiles = p.group * p.mt, pairs = (tiles + 1) >> 1;
    XFwdUnit u;
    int x = g.unit;
    u.tile0 = 2 * (x % pairs);
    x /= pairs;
    u.hk = x % p.hkv;
    u.b = x / p.hkv;
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
__global__ void __launch_bounds__(kAttnThreads, 1)
xattn_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                 const __grid_constant__ XFwdParams p) {
    constexpr int kAtoms = kD / 64;
    constexpr int kOperandBytes = kAtoms * kHalfBytes;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
    const uint32_t sQ = smem_u32(smem);
    const uint32_t sK = sQ + 2 * kTileBytes;
    const uint32_t sV = sK + 2 * kTileBytes;
    XFwdCtl* ctl = reinterpret_cast<XFwdCtl*>(smem + 6 * kTileBytes + 2 * kSoftmaxWarps * kXStageBytes);
    volatile int* s_abort = &ctl->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) ctl->abort = p.status != nullptr ? *reinterpret_cast<volatile int*>(p.status) : 0;
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
            mbar_init(smem_u32(&ctl->s_full[s][0]), 1);
            mbar_init(smem_u32(&ctl->s_full[s][1]), 1);
            for (int c = 0; c < kPieces; ++c) {
                mbar_init(smem_u32(&ctl->p_full[s][c]), kTileM);
                mbar_init(smem_u32(&ctl->o_done[s][c]), 1);
            }
        }
        mbar_init(smem_u32(&ctl->teardown), 1);
        mbar_init_fence();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&ctl->tmem_base), kTmemCols);
        tmem_relinquish();
    }
    if (warp == kTmaWarp && lane == 0) {
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
    if (warp == kTmaWarp) {
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
                    const int i = w.tile0 + t, g = i / p.mt;
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
    } else if (warp == kMmaWarp) {
        // =============================== MMA issuer ========================================
        constexpr uint32_t idesc_qk = make_idesc_f16(kBF16, false, kTileM, kTileN / 2);
        constexpr uint32_t idesc_pv = make_idesc_f16(kBF16, true, kTileM, kD);
        const uint32_t leader = elect_one() ? 1u : 0u;
        const uint64_t dq0 = smem_desc_sw128(sQ, 16, 1024);
        const uint64_t dv0 = smem_desc_sw128(sV, kHalfBytes, 1024);
        const uint32_t hi_qk = static_cast<uint32_t>(dq0 >> 32), hi_v = static_cast<uint32_t>(dv0 >> 32);
        const uint32_t lo_q = static_cast<uint32_t>(dq0), lo_v = static_cast<uint32_t>(dv0);
        const uint32_t lo_k = static_cast<uint32_t>(smem_desc_sw128(sK, 16, 1024));
        auto issue_qk_half = [&](int t, int st, int half) {
            const uint32_t a0 = lo_q + ((t * kTileBytes) >> 4);
            const uint32_t b0 = lo_k + ((st * kTileBytes + half * 64 * 128) >> 4);
            const uint32_t d = tmem + kColS0 + t * kTileN + half * (kTileN / 2);
#pragma unroll
            for (int ks = 0; ks < kD / 16; ++ks) {
                const uint32_t off = ((ks >> 2) * kHalfBytes + (ks & 3) * 32) >> 4;
                tc_mma_ss_elect(d, a0 + off, hi_qk, b0 + off, hi_qk, idesc_qk, ks > 0 ? 1u : 0u, leader);
            }
        };
        auto issue_pv_piece = [&](int t, int st, int piece, bool acc) {
            const uint32_t b0 = lo_v + ((st * kTileBytes) >> 4);
            const uint32_t a0 = tmem + kColS0 + t * kTileN;
            const uint32_t d = tmem + kColO0 + t * kD;
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                const int ks = piece * 2 + k2;
                tc_mma_ts_elect(d, a0 + (piece >> 1) * (kTileN / 2) + (ks & 3) * 8, b0 + ((ks * 16 * 128) >> 4), hi_v,
                                idesc_pv, (acc || ks > 0) ? 1u : 0u, leader);
            }
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
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    issue_qk_half(t, j & 1, half);
                    tc_commit_elect(smem_u32(&ctl->s_full[t][half]), leader);
                }
            tc_commit_elect(smem_u32(&ctl->k_empty[j & 1]), leader);
            if (n == 1) tc_commit_elect(smem_u32(&ctl->q_empty), leader);
            for (int i = 0; i < n && ok; ++i, ++j) {
                const int st = j & 1, stn = (j + 1) & 1;
                const bool more = i + 1 < n;
                ok = wait(p.words != nullptr ? &ctl->v_clean[st] : &ctl->v_full[st], (j >> 1) & 1);
                if (ok && more) ok = wait(&ctl->k_full[stn], ((j + 1) >> 1) & 1);
                if (!ok) break;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
#pragma unroll
                        for (int c = 2 * half; c < 2 * half + 2; ++c) {
                            ok = wait(&ctl->p_full[t][c], j & 1);
                            if (!ok) break;
                            tc_fence_after();
                            issue_pv_piece(t, st, c, i > 0);
                            tc_commit_elect(smem_u32(&ctl->o_done[t][c]), leader);
                        }
                        if (!ok) break;
                        if (half == 1 && t == 1) tc_commit_elect(smem_u32(&ctl->v_empty[st]), leader);
                        if (more) {
                            issue_qk_half(t, stn, half);
                            tc_commit_elect(smem_u32(&ctl->s_full[t][half]), leader);
                            if (half == 1 && t == 1) {
                                tc_commit_elect(smem_u32(&ctl->k_empty[stn]), leader);
                                if (i + 2 == n) tc_commit_elect(smem_u32(&ctl->q_empty), leader);
                            }
                        }
                    }
                    if (!ok) break;
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
    } else if (warp == kTmaWarp + 1 && p.words != nullptr) {
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
    } else if (warp < kSoftmaxWarps) {
        // =============================== softmax + epilogue ================================
        const int quarter = warp & 3, t = warp >> 2;
        const int row_in_tile = quarter * 32 + lane;
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t tS = tmem + lane_base + kColS0 + t * kTileN;
        const uint32_t tO = tmem + lane_base + kColO0 + t * kD;
        const float sl = p.scale_log2;
        bool ok = true;
        int j = 0;
        while (ok && cursor.next(p.sched, seg)) {
            const XFwdUnit w = x_fwd_unit(p, seg);
            const int n = w.hi - w.lo;
            const unsigned long long* mrow = p.words != nullptr ? p.words + static_cast<long long>(w.b) * n_words : nullptr;
            float m_ref = -INFINITY, l_sum = 0.f;
            uint32_t buf[2][32];
            bool pre = false;
            int pending = -1;
            for (int i = 0; i < n && ok; ++i, ++j) {
                const unsigned long long kw0 = x_key_word(mrow, p.skv, 2 * (w.lo + i));
                const unsigned long long kw1 = x_key_word(mrow, p.skv, 2 * (w.lo + i) + 1);
                const bool plain = (kw0 & kw1) == ~0ull;  // (the same for the whole CTA)
#pragma unroll
                for (int c = 0; c < kPieces; ++c) {
                    const int half = c >> 1, hc = c & 1;
                    uint32_t(&sc)[32] = buf[hc];
                    if (!pre) {
                        if (pending >= 0) {  // never block with a hand-over outstanding
                            tc_wait_st();
                            tc_fence_before();
                            mbar_arrive(smem_u32(&ctl->p_full[t][pending]));
                            pending = -1;
                        }
                        if (hc == 0) {
                            // (a vote: a wait that gives up in some lanes only must not split the warp)
                            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&ctl->s_full[t][half]), j & 1, s_abort,
                                                                   p.status, limit, PA_DEV_TIMEOUT_PIPE)) && ok;
                            tc_fence_after();
                        }
                        tmem_ld32(tS + c * kPieceCols, sc);
                    }
                    tc_wait_ld();
                    tmem_ld_fence(sc);
                    pre = false;
                    if (hc == 0) {
                        pre = true;
                    } else if (c == 1) {
                        pre = __all_sync(0xffffffffu, mbar_try_wait(smem_u32(&ctl->s_full[t][1]), j & 1));
                    } else if (i + 1 < n) {
                        pre = __all_sync(0xffffffffu, mbar_try_wait(smem_u32(&ctl->s_full[t][0]), (j + 1) & 1));
                    }
                    if (pre) {
                        if (hc == 1) tc_fence_after();
                        tmem_ld32(tS + ((c + 1) & 3) * kPieceCols, buf[hc ^ 1]);
                    }
                    uint32_t live = 0xffffffffu;
                    uint32_t pk[16];
                    float ls, mx;
                    if (c == 0 && i == 0) {
                        // A row's first logits set its reference: with few key tiles the guess from earlier pieces,
                        // which the later ones take, would be wrong once in every 16 pieces.
                        const uint32_t seen = plain ? 0xffffffffu : static_cast<uint32_t>(kw0);
#pragma unroll
                        for (int x = 0; x < 32; x += 2)
                            m_ref = fmax3(m_ref, ((seen >> x) & 1u) ? __uint_as_float(sc[x]) : -INFINITY,
                                          ((seen >> (x + 1)) & 1u) ? __uint_as_float(sc[x + 1]) : -INFINITY);
                    }
                    const float neg = (m_ref == -INFINITY) ? 0.0f : -m_ref * sl;
                    if (plain) {
                        softmax_chunk<kBF16, false>(sc, live, sl, neg, pk, ls, mx);
                    } else {
                        live = static_cast<uint32_t>((half ? kw1 : kw0) >> (hc * 32));
                        softmax_chunk<kBF16, true>(sc, live, sl, neg, pk, ls, mx);
                    }
                    if (pending >= 0) {
                        tc_wait_st();
                        tc_fence_before();
                        mbar_arrive(smem_u32(&ctl->p_full[t][pending]));
                        pending = -1;
                    }
                    const bool grow = (mx - m_ref) * sl > kRescaleThreshold;  // (-inf - -inf: NaN, false)
                    const uint32_t tP = tS + half * (kTileN / 2) + hc * (kPieceCols / 2);
                    if (__any_sync(0xffffffffu, grow)) {
                        if (pre) {
                            tc_wait_ld();
                            tmem_ld_fence(buf[hc ^ 1]);
                        }
                        const uint32_t bo = (c > 0) ? smem_u32(&ctl->o_done[t][c - 1]) : smem_u32(&ctl->o_done[t][kPieces - 1]);
                        const uint32_t par = (c > 0) ? (j & 1) : ((j - 1) & 1);
                        const float2 r = softmax_piece_regrow<kBF16, kD>(tS + c * kPieceCols, tP, tO, live, sl, mx, m_ref,
                                                                         l_sum, i > 0 || c > 0, bo, par, s_abort, p.status,
                                                                         limit);
                        m_ref = r.x;
                        l_sum = r.y;
                    } else {
                        l_sum += ls;
                        tmem_st16(tP, pk);
                    }
                    if (hc == 0) {
                        pending = c;
                    } else {
                        tc_wait_st();
                        tc_fence_before();
                        mbar_arrive(smem_u32(&ctl->p_full[t][c]));
                    }
                }
            }
            if (n > 0)
                ok = mbar_wait(smem_u32(&ctl->o_done[t][kPieces - 1]), (j - 1) & 1, s_abort, p.status, limit,
                               PA_DEV_TIMEOUT_PIPE) && ok;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const int tile = w.tile0 + t, g = tile / p.mt;
            const int row = (tile - g * p.mt) * kTileM + row_in_tile;
            const bool in_range = g < p.group && row < p.sq;
            const int head = w.hk * p.group + g;
            if (seg.slot >= 0) {
                // this CTA's share of a unit: unnormalised O, reference and row sum
                const int r256 = t * kTileM + row_in_tile;
                float4* po = reinterpret_cast<float4*>(p.part_o) + static_cast<long long>(seg.slot) * (kD / 4) * 256 + r256;
#pragma unroll
                for (int b = 0; b < kD / 32; ++b) {
                    uint32_t o[32];
                    tmem_ld32(tO + b * 32, o);
                    tc_wait_ld();
                    tmem_ld_fence(o);
                    if (n <= 0) {
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] = 0u;
                    }
#pragma unroll
                    for (int v4 = 0; v4 < 8; ++v4)
                        __stcg(po + (b * 8 + v4) * 256,
                               make_float4(__uint_as_float(o[4 * v4]), __uint_as_float(o[4 * v4 + 1]),
                                           __uint_as_float(o[4 * v4 + 2]), __uint_as_float(o[4 * v4 + 3])));
                }
                __stcg(p.part_ml + static_cast<long long>(seg.slot) * 256 + r256, make_float2(m_ref, l_sum));
                continue;
            }
            const float inv = l_sum > 0.0f ? 1.0f / l_sum : 0.0f;  // (no key at all: zeros, LSE -inf)
            uint8_t* stage = smem + 6 * kTileBytes + warp * (2 * kXStageBytes);
            const bool zero = n <= 0 || !(l_sum > 0.0f);
            const int row_w = (tile - g * p.mt) * kTileM + quarter * 32;  // first of the warp's rows
#pragma unroll
            for (int b = 0; b < kD / 32; ++b) {
                uint32_t o[32];
                tmem_ld32(tO + b * 32, o);
                if (lane == 0) tma_store_wait_read<1>();  // (this buffer's last store has been read)
                __syncwarp();
                tc_wait_ld();
                tmem_ld_fence(o);
                if (zero) {
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = 0u;
                }
                x_stage32<kBF16>(stage + (b & 1) * kXStageBytes, lane, o, inv);
                fence_proxy_async_shared();
                __syncwarp();
                if (lane == 0 && g < p.group && row_w < p.sq)
                    tma_store_5d(&tm_o, smem_u32(stage + (b & 1) * kXStageBytes), b * 32, row_w, head, w.b, 0);
            }
            if (in_range && p.lse != nullptr)
                p.lse[(static_cast<long long>(w.b) * p.hkv * p.group + head) * p.sq + row] =
                    l_sum > 0.0f ? m_ref * p.scale + logf(l_sum) : -INFINITY;
        }
        if (lane == 0) tma_store_wait();
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) x_report(p.status_host, ctl->abort);
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// Joins the partial results of units that several CTAs worked on (see XSched): one block per
// cut unit and 8 output columns, one thread per row.
//   out = sum_i 2^((m_i - m) sl) O_i / sum_i 2^((m_i - m) sl) l_i
template <bool kBF16, int kD>
__global__ void __launch_bounds__(256)
xattn_fwd_join_kernel(const __grid_constant__ XFwdParams p, int grid) {
    XCut cut;
    if (!x_cut_unit(p.sched, blockIdx.x, grid, cut)) return;
    const int unit = cut.unit, cols0 = blockIdx.y * 8, r256 = threadIdx.x;
    const float sl = p.scale_log2;
    float m = -INFINITY;
    x_for_parts(p.sched, cut, [&](int slot) { m = fmaxf(m, __ldcg(p.part_ml + static_cast<long long>(slot) * 256 + r256).x); });
    float acc[8], l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    x_for_parts(p.sched, cut, [&](int slot) {
        const float2 ml = __ldcg(p.part_ml + static_cast<long long>(slot) * 256 + r256);
        if (ml.x == -INFINITY) return;  // (a share that saw no key)
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
    const int tile = w.tile0 + (r256 >> 7), grp = tile / p.mt;
    const int row = (tile - grp * p.mt) * kTileM + (r256 & 127);
    if (grp >= p.group || row >= p.sq) return;
    const int head = w.hk * p.group + grp;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    uint16_t* orow = p.out + (w.b * p.o_sb + head * p.o_sh + row * p.o_ss) + cols0;
    uint32_t q[4];
#pragma unroll
    for (int x = 0; x < 4; ++x)
        q[x] = kBF16 ? pack_bf16x2(acc[2 * x] * inv, acc[2 * x + 1] * inv) : pack_f16x2(acc[2 * x] * inv, acc[2 * x + 1] * inv);
    *reinterpret_cast<uint4*>(orow) = make_uint4(q[0], q[1], q[2], q[3]);
    if (blockIdx.y == 0 && p.lse != nullptr)
        p.lse[(static_cast<long long>(w.b) * p.hkv * p.group + head) * p.sq + row] =
            l > 0.f ? m * p.scale + logf(l) : -INFINITY;
}

}  // namespace pa
