// libdmm, second translation unit: the operators around the product with compressed weights.
//   the product with bias, activation (plain or gated) and residual in its epilogue   dmm_decode_matmul_fused
//   the same per expert, rows grouped by expert with ragged sizes                      dmm_decode_matmul_grouped
//   the choice of experts and the lists the grouped product reads                      dmm_route_experts
//   the weighted sum of the experts' rows                                              dmm_combine_experts
// Kernels and host code in the files included below, each inside namespace dmm; the decode tables, the
// matrix-vector helpers and the matrix-matrix kernel's body are shared with dmm.hip.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <atomic>
#include <thread>
#include <type_traits>
#include <vector>
#include <hip/hip_ext.h>
#include <math.h>
#include <stdint.h>
#include <stdlib.h>

#include "dmm.h"

namespace dmm {

#include "dmm_types.h"
#include "dmm_launch.h"
#include "dmm_hostroute.h"
#include "dmm_tables.h"
#include "dmm_gemv_f16.h"
#include "dmm_gemv_q8.h"
#include "dmm_gemv_q8d.h"
#include "dmm_gemv_f16d.h"
#include "dmm_gemm.h"
#include "dmm_epilogue.h"
#include "dmm_ops_rows.h"
#include "dmm_ops_mid.h"
#include "dmm_ops_gemm.h"
#include "dmm_route.h"
#include "dmm_ops_host.h"

}  // namespace dmm

using namespace dmm;

extern "C" {

int dmm_decode_matmul_fused(const void *x, const void *codes, const void *grid, const dmm_epilogue *ep, void *y, int64_t M, int64_t N,
                            int64_t K, void *workspace, int64_t workspace_bytes, void *stream)
{
    int st = check_ops(x, M, codes, grid, ep, y, M, 1, N, K);
    if (st != DMM_OK || M == 0 || N == 0) return st;
    if (workspace_bytes < 0) return DMM_ERR_BAD_SHAPE;
    if (workspace && workspace_bytes > 0 && !aligned(workspace, 16)) return DMM_ERR_MISALIGNED;
    if ((st = ensure_ready((hipStream_t)stream))) return st;
    const Groups g{nullptr, nullptr, 1, (int)M, (int)M};
    return dispatch_ops(x, codes, grid, g, make_epi(*ep, y, N, nullptr, 1), ep->gated != 0, K, workspace, workspace_bytes,
                        (hipStream_t)stream);
}

int dmm_set_ops_kernel(int kernel)
{
    if (kernel < -1 || kernel > kOpsMid) return DMM_ERR_BAD_SHAPE;
    return g_ops_kernel.exchange(kernel, std::memory_order_relaxed);
}

int64_t dmm_fused_workspace_bytes(int64_t M, int64_t N, int64_t K, int gated) { return ops_workspace_bytes(M, N, K, gated != 0); }

static int check_grouped(const void *x, int64_t T, const void *rows, const void *codes, const void *grid, const void *scales,
                         int scale_cols, const void *offsets, const dmm_epilogue *ep, const void *y, int64_t R, int64_t E, int64_t N,
                         int64_t K)
{
    int st = check_ops(x, T, codes, grid, ep, y, R, E, N, K);
    if (st != DMM_OK) return st;
    if (ep->residual || (scales && scale_cols != 1 && !(scale_cols == 2 && ep->gated)) || (!rows && R > 0 && T != R)) return DMM_ERR_BAD_SHAPE;
    if (R == 0 || N == 0 || E == 0) return DMM_OK;
    if (!offsets) return DMM_ERR_NULL_POINTER;
    if (!aligned(offsets, 4) || !aligned(rows, 4) || !aligned(scales, 4)) return DMM_ERR_MISALIGNED;
    return DMM_OK;
}

int dmm_decode_matmul_grouped(const void *x, int64_t T, const void *rows, const void *codes, const void *grid, const void *scales,
                              int scale_cols, const void *offsets, const dmm_epilogue *ep, void *y, int64_t R, int64_t E, int64_t N,
                              int64_t K, void *stream)
{
    int st = check_grouped(x, T, rows, codes, grid, scales, scale_cols, offsets, ep, y, R, E, N, K);
    if (st != DMM_OK || R == 0 || N == 0 || E == 0) return st;
    if ((st = ensure_ready((hipStream_t)stream))) return st;
    const Groups g{(const int32_t *)offsets, (const int32_t *)rows, (int)E, (int)R, (int)T};
    return dispatch_ops(x, codes, grid, g, make_epi(*ep, y, N, (const float *)scales, scale_cols), ep->gated != 0, K, nullptr, 0,
                        (hipStream_t)stream);
}

int64_t dmm_route_workspace_bytes(int64_t T, int64_t E)
{
    if (T < 1 || T > kRouteMaxT || E < 1 || E > kRouteMaxE) return 0;
    const int64_t blocks = route_blocks(T);
    return blocks == 1 ? 0 : E * (blocks * 8 * route_words(T) + (blocks + 3) / 4 * 16);
}

int dmm_route_experts(const void *logits, int logits_type, int64_t T, int64_t E, int64_t k, int scoring, int normalize, void *weights,
                      void *experts, void *offsets, void *rows, void *slots, void *workspace, int64_t workspace_bytes, void *stream)
{
    int st = check_route(logits, logits_type, T, E, k, scoring, weights, experts, offsets, rows, slots);
    if (st != DMM_OK) return st;
    const int64_t blocks = T > 0 ? route_blocks(T) : 1, need = dmm_route_workspace_bytes(T, E);
    if (need > 0) {
        if (!workspace) return DMM_ERR_NULL_POINTER;
        if (workspace_bytes < need) return DMM_ERR_SCRATCH_TOO_SMALL;
        if (!aligned(workspace, 16)) return DMM_ERR_MISALIGNED;
    }
    if ((st = ensure_ready((hipStream_t)stream))) return st;
    RouteArgs a;
    a.logits = logits;
    a.type = logits_type;
    a.T = (int)T;
    a.E = (int)E;
    a.k = (int)k;
    a.sigmoid = scoring == DMM_SCORE_SIGMOID;
    a.normalize = normalize != 0;
    a.weights = (float *)weights;
    a.experts = (int32_t *)experts;
    a.offsets = (int32_t *)offsets;
    a.rows = (int32_t *)rows;
    a.slots = (int32_t *)slots;
    a.words = T > 0 ? route_words(T) : 1;
    a.blocks4 = (int)((blocks + 3) / 4 * 4);
    // the counts first: rows of a multiple of 16 bytes, so that the masks behind them are aligned too
    a.counts = (int32_t *)workspace;
    a.masks = blocks > 1 ? (uint64_t *)((char *)workspace + E * a.blocks4 * 4) : nullptr;
    hipStream_t s = (hipStream_t)stream;
    if (k <= 16 && E <= 256) {
        if (E <= 16) return launch_route<1, 16>(a, blocks, s);
        if (E <= 32) return launch_route<2, 16>(a, blocks, s);
        if (E <= 64) return launch_route<4, 16>(a, blocks, s);
        if (E <= 128) return launch_route<8, 16>(a, blocks, s);
        return launch_route<16, 16>(a, blocks, s);
    }
    if (E <= 64) return launch_route<1, 64>(a, blocks, s);
    if (E <= 128) return launch_route<2, 64>(a, blocks, s);
    if (E <= 256) return launch_route<4, 64>(a, blocks, s);
    if (E <= 512) return launch_route<8, 64>(a, blocks, s);
    return launch_route<16, 64>(a, blocks, s);
}

int dmm_combine_experts(const void *y, int y_type, const void *slots, const void *weights, const void *residual, int residual_type,
                        void *out, int out_type, int64_t R, int64_t T, int64_t k, int64_t N, void *stream)
{
    int st = check_combine(y, y_type, slots, weights, residual, residual_type, out, out_type, R, T, k, N);
    if (st != DMM_OK || T == 0 || N == 0) return st;
    if ((st = ensure_ready((hipStream_t)stream))) return st;
    const CombineArgs a{y, (const int32_t *)slots, (const float *)weights, residual, out, y_type == DMM_F32, residual_type == DMM_F32,
                        out_type == DMM_F32, (int)R, (int)T, (int)k, (int)N};
    const unsigned bx = (unsigned)((N + 2047) / 2048), by = (unsigned)(T < 65535 ? T : 65535);
    if (k <= 2) return launch(combine_kernel<2>, dim3(bx, by), dim3(256), 0, (hipStream_t)stream, a);
    return launch(combine_kernel<4>, dim3(bx, by), dim3(256), 0, (hipStream_t)stream, a);
}

int dmm_decode_matmul_fused_host(const void *x, const void *codes, const void *grid, const dmm_epilogue *ep, void *y, int64_t M,
                                 int64_t N, int64_t K)
{
    const int st = check_ops(x, M, codes, grid, ep, y, M, 1, N, K);
    if (st != DMM_OK || M == 0 || N == 0) return st;
    return host_ops(x, M, nullptr, codes, grid, nullptr, 1, nullptr, *ep, y, M, 1, N, K);
}

int dmm_decode_matmul_grouped_host(const void *x, int64_t T, const void *rows, const void *codes, const void *grid, const void *scales,
                                   int scale_cols, const void *offsets, const dmm_epilogue *ep, void *y, int64_t R, int64_t E, int64_t N,
                                   int64_t K)
{
    const int st = check_grouped(x, T, rows, codes, grid, scales, scale_cols, offsets, ep, y, R, E, N, K);
    if (st != DMM_OK || R == 0 || N == 0 || E == 0) return st;
    return host_ops(x, T, (const int32_t *)rows, codes, grid, (const float *)scales, scale_cols, (const int32_t *)offsets, *ep, y, R, E, N,
                    K);
}

int dmm_route_experts_host(const void *logits, int logits_type, int64_t T, int64_t E, int64_t k, int scoring, int normalize,
                           void *weights, void *experts, void *offsets, void *rows, void *slots)
{
    const int st = check_route(logits, logits_type, T, E, k, scoring, weights, experts, offsets, rows, slots);
    if (st != DMM_OK) return st;
    float *w = (float *)weights;
    int32_t *ex = (int32_t *)experts, *of = (int32_t *)offsets, *ro = (int32_t *)rows, *sl = (int32_t *)slots;
    for (int64_t e = 0; e <= E; e++) of[e] = 0;
    for (int64_t t = 0; t < T; t++) {
        bool bad = false;
        for (int64_t e = 0; e < E; e++) {
            const float v = host_load(logits, t * E + e, logits_type);
            bad = bad || v != v;
        }
        float big = 0.f, total = 0.f;
        int64_t n = 0;
        for (; n < k; n++) {   // the largest not chosen yet, lowest index first
            int best = -1;
            float bv = -INFINITY;
            for (int64_t e = 0; e < E; e++) {
                const float v = host_load(logits, t * E + e, logits_type);
                if (!(v > bv)) continue;   // equal ones later, -inf and NaN never
                bool taken = false;
                for (int64_t j = 0; j < n; j++) taken = taken || ex[t * k + j] == e;
                if (taken) continue;
                best = (int)e;
                bv = v;
            }
            if (best < 0) break;
            if (n == 0) big = bv;
            ex[t * k + n] = best;
            if (scoring != DMM_SCORE_SIGMOID) w[t * k + n] = expf(bv - big);
            else if (normalize) w[t * k + n] = expf(fminf(bv, 0.f) - fminf(big, 0.f)) / (1.f + expf(-fabsf(bv)));
            else w[t * k + n] = 1.f / (1.f + expf(-bv));
            of[best + 1]++;
        }
        if (normalize) {
            for (int64_t j = 0; j < n; j++) total += w[t * k + j];
        } else if (scoring == DMM_SCORE_SIGMOID) {
            total = 1.f;
        } else {
            for (int64_t e = 0; e < E; e++) total += expf(host_load(logits, t * E + e, logits_type) - big);
        }
        for (int64_t j = 0; j < k; j++) {
            if (j >= n) ex[t * k + j] = -1;
            w[t * k + j] = bad ? NAN : j < n ? w[t * k + j] / total : 0.f;
        }
    }
    for (int64_t e = 0; e < E; e++) of[e + 1] += of[e];
    for (int64_t i = 0; i < T * k; i++) ro[i] = sl[i] = -1;
    // a stable pass: of[e] runs through expert e's rows, and is put back afterwards
    for (int64_t i = 0; i < T * k; i++) {
        if (ex[i] < 0) continue;
        sl[i] = of[ex[i]]++;
        ro[sl[i]] = (int32_t)(i / k);
    }
    for (int64_t e = E - 1; e > 0; e--) of[e] = of[e - 1];
    of[0] = 0;
    return DMM_OK;
}

int dmm_combine_experts_host(const void *y, int y_type, const void *slots, const void *weights, const void *residual,
                             int residual_type, void *out, int out_type, int64_t R, int64_t T, int64_t k, int64_t N)
{
    const int st = check_combine(y, y_type, slots, weights, residual, residual_type, out, out_type, R, T, k, N);
    if (st != DMM_OK || T == 0 || N == 0) return st;
    const int32_t *sl = (const int32_t *)slots;
    const float *w = (const float *)weights;
    host_parallel_rows(T, (k + 1) * N, [=](int64_t t0, int64_t t1) {
        for (int64_t t = t0; t < t1; t++)
            for (int64_t n = 0; n < N; n++) {
                float acc = 0.f;
                for (int64_t j = 0; j < k; j++) {
                    const int32_t s = sl[t * k + j];
                    if (s >= 0 && s < R) acc = __builtin_fmaf(w[t * k + j], host_load(y, (int64_t)s * N + n, y_type), acc);
                }
                if (residual) acc += host_load(residual, t * N + n, residual_type);
                host_store(out, t * N + n, out_type, acc);
            }
    });
    return DMM_OK;
}

}  // extern "C"
