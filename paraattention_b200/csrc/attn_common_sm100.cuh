// What the attention kernels share: tile sizes, warp roles, and the softmax of one thread over a
// piece of 32 logits.
#pragma once
#include <cuda.h>
#include <cstdint>

#include "../../include/pa_b200.h"
#include "pa_ptx.cuh"

namespace pa {

// head_dim is a template parameter of the kernel (kD = 64 or 128). Shared-memory slots keep
// the 128-wide size for both: a 64-wide tile is one swizzle atom and fills the first half.
constexpr int kTileM = 128;
constexpr int kTileN = 128;
constexpr int kHalfBytes = 128 * 128;       // 128 rows x 64 elements x 2 B (one swizzle atom wide)
constexpr int kTileBytes = 2 * kHalfBytes;  // 128 x 128 x 2 B
constexpr int kStages = 2;
constexpr int kSoftmaxWarps = 8;
constexpr int kMmaWarp = 8;
constexpr int kTmaWarp = 9;
constexpr int kAttnThreads = 384;  // 2 softmax warpgroups + 1 control warpgroup
constexpr int kRegsLaunch = 168;   // 65536 / 384, rounded down to a multiple of 8
#ifndef PA_REGS_SOFTMAX
#define PA_REGS_SOFTMAX 168
#endif
#ifndef PA_REGS_CONTROL
#define PA_REGS_CONTROL 168
#endif
constexpr int kRegsSoftmax = PA_REGS_SOFTMAX;
constexpr int kRegsControl = PA_REGS_CONTROL;
static_assert(2 * kRegsSoftmax + kRegsControl <= 3 * kRegsLaunch, "setmaxnreg budget exceeds the launch allocation");
static_assert(kRegsSoftmax % 8 == 0 && kRegsControl % 8 == 0, "setmaxnreg counts are multiples of 8");
constexpr int kPieces = 4;         // P is handed to the tensor core in pieces of 32 key columns
constexpr int kPieceCols = kTileN / kPieces;
static_assert(kPieceCols == 32, "the softmax loads and hands over 32 columns at a time");
constexpr int kTmemCols = 512;
constexpr uint32_t kColS0 = 0, kColO0 = 256;
// log2-domain growth of the running row maximum that is tolerated before O is rescaled
constexpr float kRescaleThreshold = 8.0f;
// of every 8 pairs of probabilities, how many are exponentiated with the FMA-pipe polynomial
#ifndef PA_POLY_PAIRS_OF_8
#define PA_POLY_PAIRS_OF_8 0
#endif
constexpr int kPolyPairsOf8 = PA_POLY_PAIRS_OF_8;

// Softmax of one thread over 32 logits held in registers: p = 2^(s * sl + neg) packed to 16-bit
// pairs (pk[i] = columns 2i, 2i+1), their fp32 sum, and the largest raw logit. With kMasked, columns whose bit in
// `live` is clear count as -inf (the unmasked instantiation carries no per-element mask code at
// all: it is the one that runs on every full tile). kPolyPairsOf8 of every 8 pairs take an
// FMA-pipe polynomial instead of the special-function unit (off by default).
template <bool kBF16, bool kMasked>
__device__ __forceinline__ void softmax_chunk(const uint32_t (&sc)[32], uint32_t live, float sl, float neg,
                                              uint32_t (&pk)[16], float& sum, float& mx) {
    const float2 sl2 = make_float2(sl, sl);
    const float2 neg2 = make_float2(neg, neg);
    float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        float s0 = __uint_as_float(sc[i]), s1 = __uint_as_float(sc[i + 1]);
        if (kMasked) {
            if (((live >> i) & 1u) == 0) s0 = -INFINITY;
            if (((live >> (i + 1)) & 1u) == 0) s1 = -INFINITY;
        }
        m[(i >> 1) & 1] = fmax3(m[(i >> 1) & 1], s0, s1);
        const float2 x = __ffma2_rn(make_float2(s0, s1), sl2, neg2);
        float2 e;
        if (((i >> 1) & 7) < kPolyPairsOf8) {
            e = exp2_poly2(x);
        } else {
            e.x = ex2_approx(x.x);
            e.y = ex2_approx(x.y);
        }
        ls[(i >> 1) & 1] = __fadd2_rn(ls[(i >> 1) & 1], e);
        pk[i >> 1] = kBF16 ? pack_bf16x2(e.x, e.y) : pack_f16x2(e.x, e.y);
    }
    const float2 t = __fadd2_rn(ls[0], ls[1]);
    sum = t.x + t.y;
    mx = fmaxf(m[0], m[1]);
}

// The rare path of a softmax piece, kept out of line so that the loop every tile runs stays
// small: some row of the calling warp (all 32 lanes call) outgrew its reference `m_ref` with
// this piece's maximum `mx`. Every row moves its reference up to what it has seen; once the
// P V handed over so far has completed (`wait_o`: barrier `bo`, phase parity `par`) the warp's
// rows of O at `tO` are rescaled; the piece is reloaded from `tS_piece`, exponentiated against
// the new reference and stored to `tP`. Returns the new reference and the new row sum.
template <bool kBF16, int kD>
__device__ __noinline__ float2 softmax_piece_regrow(uint32_t tS_piece, uint32_t tP, uint32_t tO, uint32_t live, float sl,
                                                    float mx, float m_ref, float l_sum, bool wait_o, uint32_t bo,
                                                    uint32_t par, volatile int* s_abort, int* status,
                                                    unsigned long long limit_ns) {
    const float m_new = fmaxf(m_ref, mx);
    // (a row that has seen no visible key yet keeps m = -inf: scale by 1, not by NaN)
    const float alpha = (m_new == -INFINITY) ? 1.0f : ex2_approx((m_ref - m_new) * sl);
    if (wait_o) {
        mbar_wait(bo, par, s_abort, status, limit_ns, PA_DEV_TIMEOUT_PIPE);
        tc_fence_after();
#pragma unroll
        for (int b = 0; b < kD / 32; ++b) {
            uint32_t o[32];
            tmem_ld32(tO + b * 32, o);
            tc_wait_ld();
            tmem_ld_fence(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(tO + b * 32, o);
        }
        // (ordered before the next P V by the caller's wait::st / fence / arrive for this piece)
    }
    uint32_t sc[32];
    tmem_ld32(tS_piece, sc);
    tc_wait_ld();
    tmem_ld_fence(sc);
    uint32_t pk[16];
    float ls, unused;
    softmax_chunk<kBF16, true>(sc, live, sl, (m_new == -INFINITY) ? 0.0f : -m_new * sl, pk, ls, unused);
    tmem_st16(tP, pk);
    return make_float2(m_new, l_sum * alpha + ls);
}

}  // namespace pa
