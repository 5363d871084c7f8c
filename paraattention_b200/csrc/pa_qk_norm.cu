// C ABI of the per-head q/k norm with rotation: argument validation and launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "../../include/pa_b200.h"
#include "pa_host.h"
#include "qk_norm_sm100.cuh"

using pa_host::fail;
using pa_host::sm_count;

namespace {

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

int max_ctas() { return sm_count() * pa::kQkNormCtasPerSm; }

int fill(const pa_qk_norm_args* a, bool backward, pa::QkNormParams* p) {
    if (a == nullptr) return fail(PA_EINVAL, "qk_norm: args is NULL");
    if (a->batch <= 0 || a->rows <= 0) return fail(PA_EINVAL, "qk_norm: batch and rows must be positive");
    if (a->head_dim != 64 && a->head_dim != 128)
        return fail(PA_ENOTSUP, "qk_norm: head_dim %d: only 64 and 128 are built", a->head_dim);
    if (a->dtype != PA_BF16 && a->dtype != PA_F16) return fail(PA_EINVAL, "qk_norm: dtype must be PA_BF16 or PA_F16");
    if ((a->cos == nullptr) != (a->sin == nullptr)) return fail(PA_EINVAL, "qk_norm: cos and sin go together");
    if (off16(a->cos) || off16(a->sin)) return fail(PA_EINVAL, "qk_norm: cos and sin must be 16-byte aligned");
    if (a->table_row0 < 0) return fail(PA_EINVAL, "qk_norm: table_row0 must not be negative");
    if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return fail(PA_EINVAL, "qk_norm: eps must be finite and not negative");
    memset(p, 0, sizeof(*p));
    for (int i = 0; i < 2; ++i) {
        if (a->x[i] == nullptr) {
            if (i == 0) return fail(PA_EINVAL, "qk_norm: x[0] must be non-NULL");
            continue;
        }
        if (a->heads[i] <= 0) return fail(PA_EINVAL, "qk_norm: heads[%d] must be positive", i);
        if (a->y[i] == nullptr || (backward && a->dy[i] == nullptr)) return fail(PA_EINVAL, "qk_norm: tensor %d: NULL pointer", i);
        if (off16(a->x[i]) || off16(a->y[i]) || (backward && off16(a->dy[i])) || off16(a->weight[i]))
            return fail(PA_EINVAL, "qk_norm: tensor %d: base pointers must be 16-byte aligned", i);
        for (int d = 0; d < 3; ++d) {
            if (a->x_stride[i][d] % 8 || a->y_stride[i][d] % 8 || (backward && a->dy_stride[i][d] % 8))
                return fail(PA_EINVAL, "qk_norm: tensor %d: byte strides must be multiples of 16", i);
            p->x_s[i][d] = a->x_stride[i][d];
            p->y_s[i][d] = a->y_stride[i][d];
            p->dy_s[i][d] = backward ? a->dy_stride[i][d] : 0;
        }
        p->x[i] = static_cast<const uint16_t*>(a->x[i]);
        p->y[i] = static_cast<uint16_t*>(a->y[i]);
        p->dy[i] = backward ? static_cast<const uint16_t*>(a->dy[i]) : nullptr;
        p->w[i] = static_cast<const uint16_t*>(a->weight[i]);
        p->heads[i] = a->heads[i];
    }
    p->cos = a->cos;
    p->sin = a->sin;
    p->row0 = a->table_row0;
    p->batch = a->batch;
    p->rows = a->rows;
    p->eps = a->eps;
    // Shares of a row's heads: enough to occupy every warp, and such that the items fill the last round of
    // warps well (4608 rows on 2368 warps: two rounds of whole rows do the
    // work of 1.95; 2500 rows, of 1.06). A share costs about a head vector's time of its own
    // (tables, addresses), and is never less than one warp-wide access.
    const long long lines = static_cast<long long>(a->batch) * a->rows;
    const long long warps = static_cast<long long>(max_ctas()) * pa::kQkNormWarps;
    const int vec = 256 / a->head_dim;  // head vectors of one warp-wide access
    const int most = std::min((std::max(p->heads[0], p->heads[1]) + vec - 1) / vec, 4096);
    double best = 0;
    for (int c = 1; c <= most; ++c) {
        const long long rounds = (lines * c + warps - 1) / warps;
        const double turns = std::ceil(double(p->heads[0]) / c / vec) + std::ceil(double(p->heads[1]) / c / vec);
        const double t = double(rounds) * (turns + 1.0);
        if (c == 1 || t < best * 0.98) {
            best = t;
            p->chunks = c;
        }
    }
    return PA_OK;
}

template <bool kBF16, int kD, bool kBackward>
void launch(const pa::QkNormParams& p, bool adjacent, int grid, cudaStream_t s) {
    if (adjacent) pa::qk_norm_kernel<kBF16, kD, true, kBackward><<<grid, pa::kQkNormThreads, 0, s>>>(p);
    else pa::qk_norm_kernel<kBF16, kD, false, kBackward><<<grid, pa::kQkNormThreads, 0, s>>>(p);
}

template <bool kBackward>
int run(const pa_qk_norm_args* a, const pa::QkNormParams& p, int grid, cudaStream_t s) {
    const bool adjacent = a->interleaved != 0;
    if (a->dtype == PA_BF16) {
        if (a->head_dim == 128) launch<true, 128, kBackward>(p, adjacent, grid, s);
        else launch<true, 64, kBackward>(p, adjacent, grid, s);
    } else {
        if (a->head_dim == 128) launch<false, 128, kBackward>(p, adjacent, grid, s);
        else launch<false, 64, kBackward>(p, adjacent, grid, s);
    }
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(PA_ECUDA, "qk_norm launch: %s", cudaGetErrorString(e));
    return PA_OK;
}

int grid_of(const pa::QkNormParams& p) {
    const long long items = static_cast<long long>(p.batch) * p.rows * p.chunks;
    const long long ctas = (items + pa::kQkNormWarps - 1) / pa::kQkNormWarps;
    return static_cast<int>(std::min<long long>(ctas, max_ctas()));
}

}  // namespace

extern "C" {

int64_t pa_qk_norm_workspace_bytes(void) { return static_cast<int64_t>(max_ctas()) * 2 * 128 * sizeof(float); }

int pa_qk_norm_fwd(const pa_qk_norm_args* a, void* stream) {
    pa::QkNormParams p;
    const int rc = fill(a, false, &p);
    if (rc != PA_OK) return rc;
    return run<false>(a, p, grid_of(p), static_cast<cudaStream_t>(stream));
}

int pa_qk_norm_bwd(const pa_qk_norm_args* a, void* stream) {
    pa::QkNormParams p;
    int rc = fill(a, true, &p);
    if (rc != PA_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int grid = grid_of(p);
    for (int i = 0; i < 2; ++i)
        if (a->dweight[i] != nullptr && (a->weight[i] == nullptr || a->x[i] == nullptr))
            return fail(PA_EINVAL, "qk_norm: dweight[%d] without x[%d] and weight[%d]", i, i, i);
    const bool weights = a->dweight[0] != nullptr || a->dweight[1] != nullptr;
    if (weights) {
        if (a->workspace == nullptr || off16(a->workspace) ||
            a->workspace_bytes < static_cast<int64_t>(grid) * 2 * a->head_dim * static_cast<int64_t>(sizeof(float)))
            return fail(PA_EINVAL, "qk_norm: the weights' gradients need a workspace of pa_qk_norm_workspace_bytes() bytes");
        p.dw_part = static_cast<float*>(a->workspace);
    }
    rc = run<true>(a, p, grid, s);
    if (rc != PA_OK || !weights) return rc;
    uint16_t* dw[2] = {static_cast<uint16_t*>(a->dweight[0]), static_cast<uint16_t*>(a->dweight[1])};
    const dim3 block(32, 32), blocks(2 * a->head_dim / 32);
    if (a->dtype == PA_BF16) pa::qk_norm_dw_kernel<true><<<blocks, block, 0, s>>>(p.dw_part, grid, a->head_dim, dw[0], dw[1]);
    else pa::qk_norm_dw_kernel<false><<<blocks, block, 0, s>>>(p.dw_part, grid, a->head_dim, dw[0], dw[1]);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(PA_ECUDA, "qk_norm weight gradient launch: %s", cudaGetErrorString(e));
    return PA_OK;
}

}  // extern "C"
