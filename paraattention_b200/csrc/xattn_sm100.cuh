// Cross attention to an encoder's states: what the forward and the backward kernel share - how
// the work is divided over persistent CTAs, and the key mask.
//
// Queries [B, Hq, Sq, D] attend to keys / values [B or 1, Hkv, Skv, D] of another length; `group`
// = Hq / Hkv query heads share a key / value head; a boolean mask [B, Skv] drops keys.
#pragma once
#include <cstdint>

#include "attn_common_sm100.cuh"

namespace pa {

// ---- division of the work -----------------------------------------------------------------
// A kernel has `units` output tiles, each of which walks `steps` tiles of the other operand. The
// grid is one CTA per SM. Whole units (split = 0): unit u belongs to CTA u % grid, so CTAs that
// run at the same time share a head's operands in L2. Split (few units, or a poorly filled last
// round): the list of all units * steps steps is cut into equal contiguous ranges, one per CTA; a
// unit cut by a range boundary leaves fp32 partial results in a workspace slot of each CTA that
// has a part of it, and a second launch adds them in range order (results do not depend on
// scheduling). A CTA has at most one segment that begins inside a unit (slot 2 * CTA) and one
// that begins with its unit but ends inside it (slot 2 * CTA + 1).
//
// Teams (split only): where `team` consecutive units walk the same streamed tiles - the key tiles of one
// head in the backward kernel's key pass - a team of that many CTAs takes one unit each and one range
// of steps together, so that a streamed tile comes from HBM once and from L2 for the others. (Single
// ranges drift apart by a few tiles per CTA: 16380 x 512 x 40 heads read 982 MB from HBM, teams
// close to the 335 MB that q and do are.)
struct XSched {
    int units, steps, split, team;
    long long total;  // units / team * steps
};

// Division of 0 <= x < 2^31 by a constant of the launch: with l = ceil(log2 d) and m = ceil(2^(31 + l) / d), which
// is below 2^32, m d - 2^(31 + l) < d <= 2^l, so x m / 2^(31 + l) exceeds x / d by less than 1 / d. (The roles
// find their way from unit to unit with it: with the / operator the backward kernel's query pass took 478
// instead of 464 us at 32760 x 512 x 40 heads.)
struct XDiv {
    unsigned d, mul;
    int shift;
    __device__ __forceinline__ int operator()(int x) const {
        return static_cast<int>((static_cast<unsigned long long>(static_cast<unsigned>(x)) * mul) >> shift);
    }
};
inline XDiv x_div(int d) {
    XDiv v;
    int l = 0;
    while ((1ll << l) < d) ++l;
    v.d = static_cast<unsigned>(d);
    v.shift = 31 + l;
    v.mul = static_cast<unsigned>(((1ull << v.shift) + d - 1) / d);
    return v;
}

struct XSeg {
    int unit, t0, t1;
    int slot;  // -1: the whole unit is mine
};

// First step of a team's range (team = 1: a CTA's), `teams` of them in all.
__host__ __device__ inline long long x_range_begin(const XSched& s, int index, int teams) {
    return s.total * index / teams;
}
// The team whose range holds step `pos`.
__host__ __device__ inline int x_team_of(const XSched& s, long long pos, int teams) {
    int c = static_cast<int>(pos * teams / s.total);
    while (c > 0 && x_range_begin(s, c, teams) > pos) --c;
    while (c + 1 < teams && x_range_begin(s, c + 1, teams) <= pos) ++c;
    return c;
}

struct XCursor {
    int unit, stride;  // next unit; whole units: the grid, split: the team
    int t0;            // next step of it (split)
    long long left;    // steps left (split)
    __device__ __forceinline__ explicit XCursor(const XSched& s) {
        unit = blockIdx.x;
        stride = gridDim.x;
        t0 = 0;
        left = 0;
        if (s.split) {
            const int mine = blockIdx.x / s.team, teams = gridDim.x / s.team;
            const long long pos = x_range_begin(s, mine, teams);
            const int row = static_cast<int>(pos / s.steps);
            left = x_range_begin(s, mine + 1, teams) - pos;
            t0 = static_cast<int>(pos - static_cast<long long>(row) * s.steps);
            unit = row * s.team + blockIdx.x % s.team;
            stride = s.team;
        }
    }
    __device__ __forceinline__ bool next(const XSched& s, XSeg& g) {
        g.unit = unit;
        g.t0 = t0;
        g.t1 = s.steps;
        g.slot = -1;
        if (!s.split) {
            if (unit >= s.units) return false;
        } else {
            if (left <= 0) return false;
            if (left < s.steps - t0) g.t1 = t0 + static_cast<int>(left);
            if (t0 != 0 || g.t1 != s.steps) g.slot = 2 * static_cast<int>(blockIdx.x) + (t0 > 0 ? 0 : 1);
            left -= g.t1 - t0;
            t0 = 0;
        }
        unit += stride;
        return true;
    }
};

// The units that have to be joined are those that a range begins inside of, listed by the host (the joining
// kernels' blocks would spend longer on finding theirs than on the sums). No range is empty: the grid has
// at most as many teams as there are steps.
constexpr int kXMaxCtas = 160;
struct XCut {
    int unit;
    short first, last;  // teams that have a part of it
};
struct XCutList {
    int n;
    XCut cut[kXMaxCtas];
};
inline void x_list_cuts(const XSched& s, int grid, XCutList* list) {
    list->n = 0;
    const int teams = grid / s.team;
    for (int c = 1; c < teams; ++c) {
        const long long pos = x_range_begin(s, c, teams), row = pos / s.steps, a = row * s.steps;
        if (pos == a || x_range_begin(s, c - 1, teams) > a) continue;  // between units, or not the first cut of its unit
        const int last = x_team_of(s, a + s.steps - 1, teams);
        for (int m = 0; m < s.team; ++m) {
            XCut& k = list->cut[list->n++];
            k.unit = static_cast<int>(row) * s.team + m;
            k.first = static_cast<short>(c - 1);
            k.last = static_cast<short>(last);
        }
    }
}
// Calls f(slot) for the parts of a cut unit, in range order.
template <typename F>
__device__ __forceinline__ void x_for_parts(const XSched& s, const XCut& cut, F f) {
    const int member = cut.unit % s.team;
#pragma unroll 4
    for (int c = cut.first; c <= cut.last; ++c) f(2 * (c * s.team + member) + (c == cut.first ? 1 : 0));
}

// A launch in which a wait gave up tells the host, too (one thread of each CTA, at its end): the word is
// in host memory, so nobody has to copy the device's after every launch.
__device__ __forceinline__ void x_report(int* status_host, int code) {
    if (status_host != nullptr && code != 0) {
        *reinterpret_cast<volatile int*>(status_host) = code;
        __threadfence_system();
    }
}

// ---- key mask -------------------------------------------------------------------------------
// mask [B][Skv] bytes -> words[b][Skv / 64 rounded up], bit i of word w = key 64 w + i, and
// extent[b] = 1 + last key that takes part (0: none), by which the kernels skip what lies behind.
constexpr int kXMaskThreads = 256;
static __global__ void __launch_bounds__(kXMaskThreads)
xattn_mask_kernel(const uint8_t* __restrict__ mask, long long batch_stride, int keys,
                  unsigned long long* __restrict__ words, int* __restrict__ extent) {
    __shared__ int last[kXMaskThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = (keys + 63) / 64;
    const uint8_t* src = mask + blockIdx.x * batch_stride;
    unsigned long long* dst = words + static_cast<long long>(blockIdx.x) * n;
    int mine = 0;
    for (int w = warp; w < n; w += kXMaskThreads / 32) {
        const int k = w * 64 + lane;
        const unsigned lo = __ballot_sync(0xffffffffu, k < keys && src[k] != 0);
        const unsigned hi = __ballot_sync(0xffffffffu, k + 32 < keys && src[k + 32] != 0);
        if (lane == 0) dst[w] = lo | (static_cast<unsigned long long>(hi) << 32);
        if (hi != 0) mine = w * 64 + 64 - __clz(hi);
        else if (lo != 0) mine = w * 64 + 32 - __clz(lo);
    }
    if (lane == 0) last[warp] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 1; i < kXMaskThreads / 32; ++i) mine = max(mine, last[i]);
        extent[blockIdx.x] = mine;
    }
}

// The word of keys [64 block, 64 block + 64): those that exist and that the mask keeps.
__device__ __forceinline__ unsigned long long x_key_word(const unsigned long long* words, int keys, int block) {
    const int k0 = block * 64;
    if (k0 >= keys) return 0ull;
    if (words != nullptr) return __ldg(words + (k0 >> 6));
    const int n = keys - k0;
    return n >= 64 ? ~0ull : (1ull << n) - 1ull;
}

// Zeroes the rows of a loaded block of 64 keys or values (clear bit of `word` = row is masked) in shared
// memory; `base`: its first row, 64-element swizzle atoms atom_stride bytes apart. The products with
// masked rows are multiplied by zero weights; this keeps infinities and NaN that such rows may hold
// out of the sums. One whole warp calls.
template <int kD>
__device__ __forceinline__ void x_zero_rows(uint8_t* base, int atom_stride, unsigned long long word, int lane) {
    constexpr int kChunks = kD / 8;  // 16-byte chunks per row
    constexpr int kRows = 32 / kChunks;
    const int chunk = lane % kChunks;
    uint8_t* at = base + (chunk / 8) * atom_stride + (chunk % 8) * 16;
    for (int r = lane / kChunks; r < 64; r += kRows)
        if (((word >> r) & 1ull) == 0) *reinterpret_cast<uint4*>(at + r * 128) = make_uint4(0, 0, 0, 0);
}

// Writes 32 rows x 32 columns of results, one row per lane (`o`: the fp32 values of the lane's row, scaled
// by f) as 16-bit values to 2 KB of shared memory in the 64-byte swizzle of a tensor map with boxes of 32
// x 32, from where one lane stores them with TMA: the 32 lanes hold 32 different rows, so storing from
// registers touches 32 lines per instruction (measured in the forward kernel: 8700 cycles for a
// 128 x 128 tile per warpgroup, against 2950 with TMA stores from one 4 KB buffer per warp).
template <bool kBF16>
__device__ __forceinline__ void x_stage32(uint8_t* stage, int lane, const uint32_t (&o)[32], float f) {
#pragma unroll
    for (int v4 = 0; v4 < 4; ++v4) {
        uint32_t q[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float a = __uint_as_float(o[v4 * 8 + 2 * x]) * f, b = __uint_as_float(o[v4 * 8 + 2 * x + 1]) * f;
            q[x] = kBF16 ? pack_bf16x2(a, b) : pack_f16x2(a, b);
        }
        *reinterpret_cast<uint4*>(stage + lane * 64 + ((v4 ^ ((lane >> 1) & 3)) << 4)) = make_uint4(q[0], q[1], q[2], q[3]);
    }
}
constexpr int kXStageBytes = 32 * 64;

}  // namespace pa
