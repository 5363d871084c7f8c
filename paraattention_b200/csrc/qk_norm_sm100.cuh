// Per-head RMSNorm of queries and keys with the position rotation in the same pass, and its
// backward pass. Forward, for every (batch, row, head) vector x of head_dim D:
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = R (w * n)
// with R the rotation of the row's position (pairs of adjacent elements, or element i with
// i + D/2). Backward, from dy:
//   u = R^T dy,  dw = sum_{batch,row,head} u * n,  g = u * w,  dx = r (g - n mean(g * n)).
// Without a weight there is no norm (n = x, dx = u): the rotation alone.
//
// Everything is held in fp32 and rounded once, at the store. x is read again by the backward
// pass (r and n are recomputed), nothing is saved for it.
//
// HBM-bound: forward moves 4 bytes per element, backward 6. A lane owns 8 consecutive elements
// (one 16-byte access), D / 8 lanes own a vector, so a warp works on 2 (D = 128) or 4 (D = 64)
// heads of one row at a time, and the next turn's loads are issued before the last turn's
// arithmetic. A warp keeps the row's cos / sin (fp32, 16 registers) and the weights across the heads it
// works on: re-reading the tables for every head would move four times as many bytes through L1 as the
// data itself. An item of work is a row and a share of its heads of q, then of k; the host chooses how
// many shares so that the items fill whole rounds of warps.
//
// The weight gradients are summed in registers by each lane over all its heads and rows, then
// over the CTA in a fixed order; a second small kernel adds the CTAs' partial sums in a fixed
// order, so results do not depend on scheduling (no atomics).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "fbc_sm100.cuh"  // lo16 / hi16 / pack16

namespace pa {

constexpr int kQkNormThreads = 256;
constexpr int kQkNormWarps = kQkNormThreads / 32;
// Resident CTAs per SM and vectors per lane and turn, by measurement (32760 rows of 80 heads of 128): forward 243 us
// with 2 and 4 (250 with 3 and 2, 284 with 4 and 1), backward, whose weight gradients and second input
// take registers, 383 us with 2 and 2 (405 with 2 and 3, 431 with 3 and 1, 556 with 1 and 4).
constexpr int kQkNormCtasPerSm = 2;

struct QkNormParams {
    const uint16_t* x[2];   // q, k (k may be NULL)
    const uint16_t* dy[2];  // backward: gradients of the outputs
    uint16_t* y[2];         // forward: outputs; backward: dx
    long long x_s[2][3], dy_s[2][3], y_s[2][3];  // element strides (batch, row, head)
    const uint16_t* w[2];
    const float* cos;       // [>= row0 + rows][D] fp32, or NULL
    const float* sin;
    long long row0;
    int batch, rows, heads[2];
    int chunks;             // warps that share a row's heads
    float eps;
    float* dw_part;         // backward: [CTAs][2][D], or NULL
};

// Rotates the 8 elements of a lane in place (kBack: by the transpose). Half-split pairs live in
// lanes l and l ^ (D / 16) of the same vector.
template <int kD, bool kAdjacent, bool kBack>
__device__ __forceinline__ void rotate8(float (&v)[8], const float (&cs)[8], const float (&sn)[8], bool upper) {
    if constexpr (kAdjacent) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float a = v[i], c = v[i + 1];
            if constexpr (!kBack) {
                v[i] = a * cs[i] - c * sn[i];
                v[i + 1] = c * cs[i + 1] + a * sn[i + 1];
            } else {
                v[i] = a * cs[i] + c * sn[i + 1];
                v[i + 1] = c * cs[i + 1] - a * sn[i];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // forward: the lower half adds -sin * partner, the upper half + sin * partner, each with
            // its own sin; the transpose takes the partner's product with the partner's sin
            const float mine = kBack ? v[i] * sn[i] : v[i];
            const float other = __shfl_xor_sync(0xffffffffu, mine, kD / 16);
            const float turn = kBack ? (upper ? -other : other) : (upper ? other * sn[i] : -other * sn[i]);
            v[i] = v[i] * cs[i] + turn;
        }
    }
}

template <bool kBF16>
__device__ __forceinline__ void unpack8(const uint4& r, float (&v)[8]) {
    v[0] = lo16<kBF16>(r.x); v[1] = hi16<kBF16>(r.x);
    v[2] = lo16<kBF16>(r.y); v[3] = hi16<kBF16>(r.y);
    v[4] = lo16<kBF16>(r.z); v[5] = hi16<kBF16>(r.z);
    v[6] = lo16<kBF16>(r.w); v[7] = hi16<kBF16>(r.w);
}
template <bool kBF16>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    return make_uint4(pack16<kBF16>(v[0], v[1]), pack16<kBF16>(v[2], v[3]), pack16<kBF16>(v[4], v[5]),
                      pack16<kBF16>(v[6], v[7]));
}
template <int kLanes>
__device__ __forceinline__ float group_sum(float s) {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

template <bool kBF16, int kD, bool kAdjacent, bool kBackward>
__global__ void __launch_bounds__(kQkNormThreads, kQkNormCtasPerSm)
qk_norm_kernel(const __grid_constant__ QkNormParams p) {
    constexpr int kLanes = kD / 8;       // lanes per vector
    constexpr int kVec = 32 / kLanes;    // vectors a warp works on at a time
    constexpr int kUnroll = kBackward ? 2 : 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane / kLanes, at = (lane % kLanes) * 8;
    const bool upper = at >= kD / 2;

    float acc[2][8];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[t][i] = 0.f;
    uint4 w_raw[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
        w_raw[t] = p.w[t] != nullptr ? __ldg(reinterpret_cast<const uint4*>(p.w[t] + at)) : make_uint4(0, 0, 0, 0);

    const long long items = static_cast<long long>(p.batch) * p.rows * p.chunks;
    const long long stride = static_cast<long long>(gridDim.x) * kQkNormWarps;
    for (long long item = static_cast<long long>(blockIdx.x) * kQkNormWarps + warp; item < items; item += stride) {
        const int chunk = static_cast<int>(item % p.chunks);
        const long long line = item / p.chunks;
        const int row = static_cast<int>(line % p.rows);
        const int b = static_cast<int>(line / p.rows);
        float cs[8], sn[8];
        if (p.cos != nullptr) {
            const long long off = (p.row0 + row) * kD + at;
            const float4 c0 = __ldg(reinterpret_cast<const float4*>(p.cos + off));
            const float4 c1 = __ldg(reinterpret_cast<const float4*>(p.cos + off + 4));
            const float4 s0 = __ldg(reinterpret_cast<const float4*>(p.sin + off));
            const float4 s1 = __ldg(reinterpret_cast<const float4*>(p.sin + off + 4));
            cs[0] = c0.x; cs[1] = c0.y; cs[2] = c0.z; cs[3] = c0.w; cs[4] = c1.x; cs[5] = c1.y; cs[6] = c1.z; cs[7] = c1.w;
            sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w; sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) { cs[i] = 1.f; sn[i] = 0.f; }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (p.x[t] == nullptr) continue;
            const int h0 = static_cast<int>(static_cast<long long>(p.heads[t]) * chunk / p.chunks);
            const int h1 = static_cast<int>(static_cast<long long>(p.heads[t]) * (chunk + 1) / p.chunks);
            const bool normed = p.w[t] != nullptr;
            const uint16_t* xb = p.x[t] + b * p.x_s[t][0] + row * p.x_s[t][1] + at;
            const uint16_t* gb = kBackward ? p.dy[t] + b * p.dy_s[t][0] + row * p.dy_s[t][1] + at : nullptr;
            uint16_t* yb = p.y[t] + b * p.y_s[t][0] + row * p.y_s[t][1] + at;
            // (kUnroll vectors per lane in flight while as many are worked on)
            uint4 xr[kUnroll], gr[kUnroll];
            auto fetch = [&](int base) {
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    const int h = base + u * kVec + sub;
                    if (h < h1) {
                        xr[u] = __ldcs(reinterpret_cast<const uint4*>(xb + h * p.x_s[t][2]));
                        if (kBackward) gr[u] = __ldcs(reinterpret_cast<const uint4*>(gb + h * p.dy_s[t][2]));
                    }
                }
            };
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) xr[u] = gr[u] = make_uint4(0, 0, 0, 0);
            fetch(h0);
            for (int base = h0; base < h1; base += kVec * kUnroll) {
                uint4 xc[kUnroll], gc[kUnroll];
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    xc[u] = xr[u];
                    gc[u] = gr[u];
                }
                fetch(base + kVec * kUnroll);
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    if (base + u * kVec >= h1) break;  // (the same for the whole warp)
                    const int h = base + u * kVec + sub;
                    const bool live = h < h1;
                    float x[8], w[8];
                    unpack8<kBF16>(xc[u], x);
                    unpack8<kBF16>(w_raw[t], w);
                    float r = 1.f;
                    if (normed) {
                        float ss = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
                        r = rsqrtf(group_sum<kLanes>(ss) * (1.0f / kD) + p.eps);
                    }
                    float o[8];
                    if constexpr (!kBackward) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) o[i] = normed ? x[i] * r * w[i] : x[i];
                        rotate8<kD, kAdjacent, false>(o, cs, sn, upper);
                    } else {
                        unpack8<kBF16>(gc[u], o);
                        rotate8<kD, kAdjacent, true>(o, cs, sn, upper);
                        if (normed) {
                            float dot = 0.f;
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                x[i] *= r;  // n
                                // (a lane behind the last head holds the values of an earlier one)
                                acc[t][i] += live ? o[i] * x[i] : 0.f;
                                o[i] *= w[i];
                                dot = fmaf(o[i], x[i], dot);
                            }
                            dot = group_sum<kLanes>(dot) * (1.0f / kD);
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = r * (o[i] - x[i] * dot);
                        }
                    }
                    if (live) __stcs(reinterpret_cast<uint4*>(yb + h * p.y_s[t][2]), pack8<kBF16>(o));
                }
            }
        }
    }
    if constexpr (kBackward) {
        if (p.dw_part == nullptr) return;
        __shared__ float sh[kQkNormWarps * kVec][2][kD];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) sh[warp * kVec + sub][t][at + i] = acc[t][i];
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * kD; c += kQkNormThreads) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < kQkNormWarps * kVec; ++k) s += sh[k][c / kD][c % kD];
            p.dw_part[static_cast<long long>(blockIdx.x) * 2 * kD + c] = s;
        }
    }
}

// dw[t][c] = sum over CTAs of dw_part[cta][t][c], rounded to the weights' type. One block per 32
// channels; 32 threads along the CTAs' axis per channel, combined in a fixed order.
template <bool kBF16>
__global__ void __launch_bounds__(1024)
qk_norm_dw_kernel(const float* __restrict__ part, int ctas, int d, uint16_t* dwq, uint16_t* dwk) {
    __shared__ float sh[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x;  // channel of [2][d]
    float s = 0.f;
    for (int k = threadIdx.y; k < ctas; k += 32) s += __ldg(part + static_cast<long long>(k) * 2 * d + c);
    sh[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) t += sh[k][threadIdx.x];
        uint16_t* out = c < d ? dwq : dwk;
        if (out != nullptr) out[c < d ? c : c - d] = static_cast<uint16_t>(pack16<kBF16>(t, 0.f) & 0xffffu);
    }
}

}  // namespace pa
