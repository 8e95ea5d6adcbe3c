// The host side of the operators around the product: checks, dispatch, and the same operators on host memory.
// Part of libdmm: included by dmm_ops.hip inside namespace dmm; not a translation unit of its own.

inline bool type_ok(int t) { return t == DMM_F16 || t == DMM_F32; }
inline uintptr_t type_bytes(int t) { return t == DMM_F32 ? 4 : 2; }

// rows of x and of y in one call: row numbers of a tile that begins at the last row stay below 2^31
constexpr int64_t kOpsMaxRows = 1 << 30;

// Residual and output, n elements each: the same memory, element for element, or none in common.  (A half residual and a
// float output at one address would overwrite elements that are still to be read.)
inline bool residual_ok(const void *residual, int residual_type, const void *y, int out_type, int64_t n)
{
    if (!residual || (residual == y && residual_type == out_type)) return true;
    const uintptr_t r = reinterpret_cast<uintptr_t>(residual), o = reinterpret_cast<uintptr_t>(y);
    return r + (uintptr_t)n * type_bytes(residual_type) <= o || o + (uintptr_t)n * type_bytes(out_type) <= r;
}

// what both products ask of their arguments: T rows of x, R rows of y, E matrices
int check_ops(const void *x, int64_t T, const void *codes, const void *grid, const dmm_epilogue *ep, const void *y, int64_t R,
              int64_t E, int64_t N, int64_t K)
{
    if (!ep) return DMM_ERR_NULL_POINTER;
    if (T < 0 || R < 0 || E < 0 || N < 0 || K < 0 || (K & 7)) return DMM_ERR_BAD_SHAPE;
    if (ep->activation < DMM_ACT_NONE || ep->activation > DMM_ACT_GELU_TANH || !type_ok(ep->out_type) ||
        (ep->bias && !type_ok(ep->bias_type)) || (ep->residual && !type_ok(ep->residual_type)))
        return DMM_ERR_BAD_SHAPE;
    if (R == 0 || N == 0 || E == 0) return DMM_OK;
    if (!y || !grid) return DMM_ERR_NULL_POINTER;
    if (K > 0 && (!codes || (T > 0 && !x))) return DMM_ERR_NULL_POINTER;
    if (!aligned(x, 2) || !aligned(codes, 2) || !aligned(grid, 2) || !aligned(y, type_bytes(ep->out_type)) ||
        (ep->bias && !aligned(ep->bias, type_bytes(ep->bias_type))) ||
        (ep->residual && !aligned(ep->residual, type_bytes(ep->residual_type))))
        return DMM_ERR_MISALIGNED;
    if (T > kOpsMaxRows || R > kOpsMaxRows || E > 65535 || N > INT32_MAX / 2 || K > INT32_MAX) return DMM_ERR_TOO_LARGE;
    if (!residual_ok(ep->residual, ep->residual_type, y, ep->out_type, R * N)) return DMM_ERR_OVERLAP;
    return DMM_OK;
}

Epi make_epi(const dmm_epilogue &ep, void *y, int64_t N, const float *scales, int scale_cols)
{
    Epi e;
    e.bias = ep.bias;
    e.residual = ep.residual;
    e.y = y;
    e.scales = scales;
    e.scale = ep.scale;
    e.scale_up = ep.scale_up;
    e.N = (int)N;
    e.act = ep.activation;
    e.scale_cols = scale_cols;
    e.bias_f32 = ep.bias_type == DMM_F32;
    e.residual_f32 = ep.residual_type == DMM_F32;
    e.out_f32 = ep.out_type == DMM_F32;
    return e;
}

template <bool kGated>
int run_ops_generic(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, hipStream_t s)
{
    int64_t blocks = ((int64_t)e.N + 3) / 4;
    if (blocks > 65535 * 16) blocks = 65535 * 16;
    return launch(ops_generic_kernel<kGated>, dim3((unsigned)blocks, (unsigned)g.E), dim3(256), 0, s, (const uint16_t *)x,
                  (const uint16_t *)codes, grid, g, e, K);
}

// the matrix unit's kernels: 16-byte loads at 4-byte aligned places, 31-bit offsets into one expert's codes
bool ops_mfma_ok(const void *x, const void *codes, const void *grid, const Groups &g, int64_t rows, int64_t K)
{
    return K >= 16 && (K & 15) == 0 && aligned(x, 16) && aligned(codes, 16) && aligned(grid, 16) && g.T > 0 &&
           rows * (K >> 2) < (1LL << 31) && rows <= 65535LL * 128;
}

// and into x: all of them where x is below 2 GiB; the matrix-matrix kernel has its offsets from the first of up to 128 rows
// of a block if these follow each other (139266 rows of 8192, past 2 GiB, to 2048: 5.4 ms, the catch-all 760)
inline bool ops_x_near(const Groups &g, int64_t K) { return (int64_t)g.T * K * 2 < (1LL << 31); }
inline bool ops_x_by_block(const Groups &g, int64_t K) { return !g.rows && 128 * K * 2 < (1LL << 31); }

template <int TM, bool kGated>
int launch_ops_gemm(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, hipStream_t s)
{
    constexpr int BM = 32 * TM, BN = GemmOpsPlace<kGated>::kOutN;
    const int64_t tiles = ((int64_t)g.R + BM - 1) / BM + (g.offsets ? g.E : 0);   // an expert adds at most one cut tile
    return launch(ops_gemm_kernel<TM, kGated>, dim3((unsigned)tiles, (unsigned)((e.N + BN - 1) / BN)), dim3(256), gr_smem_bytes(TM), s,
                  (const uint16_t *)x, (const uint16_t *)codes, grid, g, e, (int)K);
}

// rows of y per block by the rows an expert has on average
template <bool kGated>
int run_ops_gemm(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, hipStream_t s)
{
    switch (gemm_reg_tm(g.R / g.E)) {
        case 1: return launch_ops_gemm<1, kGated>(x, codes, grid, g, e, K, s);
        case 2: return launch_ops_gemm<2, kGated>(x, codes, grid, g, e, K, s);
        default: return launch_ops_gemm<4, kGated>(x, codes, grid, g, e, K, s);
    }
}

// dmm_set_ops_kernel: what a test or a benchmark forces instead of the choice below (-1: nothing)
std::atomic<int> g_ops_kernel{-1};
enum OpsKernel { kOpsGeneric = 0, kOpsRows = 1, kOpsGemm = 2, kOpsSplit = 3, kOpsRows8 = 4, kOpsMid = 5 };

template <int NT, int XI, int W, int CG, bool kGated, bool kOne, int D = 2>
int launch_ops_rows_inst(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, int64_t units,
                         hipStream_t s)
{
    const int64_t wgs = units < cu_count() ? units : cu_count();
    const OpsRowsArgs args{(const uint16_t *)x, (const uint16_t *)codes, grid, g, e, (int)K, (int)(units / wgs), (int)(units % wgs)};
    return launch(ops_rows_kernel<NT, D, XI, W, CG, kGated, kOne>, dim3((unsigned)wgs), dim3(64 * W), (size_t)fd_lds_bytes(XI, W), s, args);
}

// most segments the rows can make, sr rows each: an expert adds at most one cut one, and none without a row
inline int64_t ops_segments(const Groups &g, int64_t sr)
{
    const int64_t full = ((int64_t)g.R + sr - 1) / sr;
    return g.offsets ? std::min<int64_t>((int64_t)g.R, (int64_t)g.R / sr + g.E) : full;
}

// Whether the jobs of a call can be counted in 31 bits, whatever the list of the experts' rows holds: one that does
// not increase may give every expert all rows.
inline bool ops_jobs_fit(const Groups &g, int64_t sr, int64_t N)
{
    return (g.offsets ? (int64_t)g.E : 1) * (((int64_t)g.R + sr - 1) / sr) * ((N + 15) / 16) < (1LL << 31);
}

// A job that 8-bit operands cannot do is done again in 16 bits, by number up to the 32nd of a workgroup's; the ones behind it
// share a bit, so that some are stored twice.  That changes nothing, except where the residual is the output itself: it
// would be added twice.  Whether no workgroup has more jobs than numbers (a job is one unit or more).
inline bool ops_redo_by_number(const Groups &g, int64_t N, int64_t cus)
{
    return ops_segments(g, 2) * ((N + 15) / 16) <= 32 * cus;
}

template <int XI, int W, int CG, bool kGated>
int launch_ops_rows(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, hipStream_t s)
{
    const int64_t units = ops_segments(g, 2 * XI * CG) * ((e.N + 15) / 16);
    const int64_t cus = cu_count(), share = (units + cus - 1) / cus * (kGated ? 2 : 1);   // most tiles a workgroup gets
    if (!g.offsets && g.R <= 2 * XI * CG && share <= 8) {
        if (share <= 2) return launch_ops_rows_inst<2, XI, W, CG, kGated, true>(x, codes, grid, g, e, K, units, s);
        if (share <= 4) return launch_ops_rows_inst<4, XI, W, CG, kGated, true>(x, codes, grid, g, e, K, units, s);
        return launch_ops_rows_inst<8, XI, W, CG, kGated, true>(x, codes, grid, g, e, K, units, s);
    }
    if constexpr (XI != 4) {   // four to eight rows: dense, one segment; not here with so few tiles
        if (share <= 2) return launch_ops_rows_inst<2, XI, W, CG, kGated, false>(x, codes, grid, g, e, K, units, s);
        if (share <= 4) return launch_ops_rows_inst<4, XI, W, CG, kGated, false>(x, codes, grid, g, e, K, units, s);
    }
    // Eight waves, gated: four code loads in flight per wave where a job has more than one step per wave (2 x 11008 x 4096, 8
    // experts, 40 rows 58.5 us with two, 54.6 with four; but 2 x 1408 x 2048, 64 experts, 128 rows 27.5 / 29.2; not gated no difference)
    if constexpr (kGated && W == 8 && CG == 1)
        if (K > 2048) return launch_ops_rows_inst<8, XI, W, CG, kGated, false, 4>(x, codes, grid, g, e, K, units, s);
    return launch_ops_rows_inst<8, XI, W, CG, kGated, false>(x, codes, grid, g, e, K, units, s);
}

template <int NT, bool kGated, bool kOne>
int launch_ops_rows8_inst(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, int64_t units,
                          hipStream_t s)
{
    const int64_t wgs = units < cu_count() ? units : cu_count();
    const OpsRowsArgs args{(const uint16_t *)x, (const uint16_t *)codes, grid, g, e, (int)K, (int)(units / wgs), (int)(units % wgs)};
    return launch(ops_rows8_kernel<NT, 2, kGated, kOne>, dim3((unsigned)wgs), dim3(1024), (size_t)kO8Bytes, s, args);
}

// 8-bit operands, two rows per segment
template <bool kGated>
int run_ops_rows8(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, hipStream_t s)
{
    const int64_t units = ops_segments(g, 2) * ((e.N + 15) / 16);
    const int64_t cus = cu_count(), share = (units + cus - 1) / cus * (kGated ? 2 : 1);
    if (!g.offsets && g.R <= 2 && share <= 8) {
        if (share <= 2) return launch_ops_rows8_inst<2, kGated, true>(x, codes, grid, g, e, K, units, s);
        if (share <= 4) return launch_ops_rows8_inst<4, kGated, true>(x, codes, grid, g, e, K, units, s);
        return launch_ops_rows8_inst<8, kGated, true>(x, codes, grid, g, e, K, units, s);
    }
    if (share <= 4) return launch_ops_rows8_inst<4, kGated, false>(x, codes, grid, g, e, K, units, s);
    return launch_ops_rows8_inst<8, kGated, false>(x, codes, grid, g, e, K, units, s);
}

inline int64_t ops_stream_lds(int64_t K) { return (int64_t)kSTablesBytes + stream_red_bytes(1, 16, 1) + stream_x_bytes(1, K); }

int launch_ops_stream(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, hipStream_t s)
{
    const int64_t tiles = ((int64_t)e.N + 15) / 16;   // one per workgroup
    const OpsRowsArgs args{(const uint16_t *)x, (const uint16_t *)codes, grid, g, e, (int)K, 1, 0};
    return launch(ops_stream_kernel, dim3((unsigned)tiles), dim3(1024), (size_t)ops_stream_lds(K), s, args);
}

// tens of rows per expert, 32 per segment
template <bool kGated>
int launch_ops_mid(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, hipStream_t s)
{
    const int64_t units = ops_segments(g, kMidRows) * ((e.N + 15) / 16);
    const int64_t wgs = units < cu_count() ? units : cu_count();
    const OpsRowsArgs args{(const uint16_t *)x, (const uint16_t *)codes, grid, g, e, (int)K, 0, 0};
    return launch(ops_mid_kernel<4, kGated>, dim3((unsigned)wgs), dim3(64 * kMidW), (size_t)kMidBytes, s, args);
}

template <int NT, int D, bool kGated>
int launch_ops_q8d_inst(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, int64_t units,
                        hipStream_t s)
{
    const int64_t wgs = units < cu_count() ? units : cu_count();
    const int64_t lds = std::max<int64_t>(qd_lds_bytes(), fd_lds_bytes(2));   // its own, and the 16-bit body's
    const OpsRowsArgs args{(const uint16_t *)x, (const uint16_t *)codes, grid, g, e, (int)K, (int)(units / wgs), (int)(units % wgs)};
    return launch(ops_q8d_kernel<NT, 1, D, kGated>, dim3((unsigned)wgs), dim3(1024), (size_t)lds, s, args);
}

inline int64_t ops_share(int64_t N, bool gated)   // most tiles a workgroup gets of one row's matrix
{
    const int64_t units = (N + 15) / 16, cus = cu_count();
    return (units + cus - 1) / cus * (gated ? 2 : 1);
}

template <bool kGated>
int launch_ops_q8d(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, hipStream_t s)
{
    const int64_t units = ((int64_t)e.N + 15) / 16;
    switch (ops_share(e.N, kGated)) {
        case 1:
        case 2: return launch_ops_q8d_inst<2, 2, kGated>(x, codes, grid, g, e, K, units, s);
        case 3:
        case 4: return launch_ops_q8d_inst<4, 2, kGated>(x, codes, grid, g, e, K, units, s);
        case 5:
        case 6: return launch_ops_q8d_inst<6, 3, kGated>(x, codes, grid, g, e, K, units, s);
        default: return launch_ops_q8d_inst<8, 2, kGated>(x, codes, grid, g, e, K, units, s);
    }
}

// Rows of a segment, and waves.  Dense: as many rows as there are.  By expert, where only the average is known: sixteen rows on
// eight waves, except for less than one row per expert on a long K (graph launches, us, four rows on sixteen waves / sixteen
// on eight: 2 x 11008 x 4096, 8 experts, 4 rows 20.6 / 21.6, 8 rows 32.9 / 33.3, 32 rows 81.7 / 58.0; 4096 x 11008, 16 experts, 4 rows
// 13.0 / 16.2, 16 rows 32.7 / 27.8; 2 x 1408 x 2048, 64 experts, 16 rows 17.1 / 15.3, 256 rows 58.4 / 33.4; eight rows on sixteen
// waves are behind one or the other).  Up to 2048 k there are no more than eight steps: half of sixteen waves would have none.
// 32 rows per segment where an expert has more than sixteen.
template <bool kGated>
int run_ops_rows(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, hipStream_t s)
{
    const bool short_k = K <= 2048;
    if (g.offsets ? g.R > 16 * (int64_t)g.E : g.R > 16) return launch_ops_rows<8, 8, 2, kGated>(x, codes, grid, g, e, K, s);
    if (!short_k && (g.R <= 4 || (g.offsets && g.R < g.E && K >= 4096))) return launch_ops_rows<2, 16, 1, kGated>(x, codes, grid, g, e, K, s);
    if (!short_k && !g.offsets && g.R <= 8) return launch_ops_rows<4, 16, 1, kGated>(x, codes, grid, g, e, K, s);
    return launch_ops_rows<8, 8, 1, kGated>(x, codes, grid, g, e, K, s);
}

// Estimates, in us, for segments of 32 rows (`segs` of them), N columns of y and K:
// the kernel for tens of rows: 5 and, per 256 k, by the tiles that a wave has on average (0.25 tiles 0.7, 0.9 tiles 0.9, 2.4 tiles
// 1.6 to 1.8, 4.4 tiles 3.0, 9 tiles 6.6);
inline double ops_mid_cost(double segs, int64_t N, int64_t K, bool gated, int cus)
{
    const double f = segs * (double)((N + 15) / 16) / (8.0 * cus);
    return 5.0 + std::max(0.6, std::max(0.2 + 0.65 * f, 0.75 * f - 0.3)) * (gated ? 2.0 : 1.0) * (double)((K + 255) / 256);
}
// the matrix-matrix kernel: 15 and K * 12 ns per round of blocks (`tiles` of 128 rows).
inline double ops_gemm_cost(double tiles, int64_t N, int64_t K, bool gated, int cus)
{
    const double blocks = tiles * (double)(((gated ? 2 * N : N) + 255) / 256), rounds = (double)(int64_t)(blocks / cus + 0.999);
    return rounds * (15.0 + (double)K * 12e-3);
}

// Dense calls of more than 32 rows: the few-rows kernel (32 rows per segment), the one for tens of rows, or split K / the
// matrix-matrix kernel (kOpsGemm stands for both).  The first costs about 7 us, K * 0.34 ns (0.5 past 512 rows, where a
// workgroup meets many segments) per 16-row tile of the busiest workgroup and 3.5 us for every eight of them after the first; the
// split what passes_beat_splitk says up to 512 rows, 14 us + 0.085 per row + 0.3 per MB of codes, and 16 us and 1 PF/s past them
// (graph launches, us, few rows / tens / split: 4096 x 4096 M = 100 12.9 / 16.6 / 25.0, 400 31.9 / 27.5 / 31.4; 4096 x 11008 M = 200 36.5 / 44.1 / 34.8;
// 2 x 137 x 11776 M = 528 24.5 / 51.3 / 49.3; 4096 x 512 M = 800 33.8 / 13.1 / 23.9; 1024 x 1024 M = 1024 12.1 / 9.2 / 22.3; 2 x 640 x
// 768 M = 1500 20.9 / 10.2 / 23.7; 104 x 320 M = 2957 8.9 / 6.5 / 22.2; 256 x 4096 M = 4096 26.6 / 23.7 / 27.8; 1024 x 4096 M = 2048 44.3 /
// 31.4 / 33.5; 2 x 11008 x 4096 M = 400 137 / 100 / 110, M = 600 198 / 154 / 116).
inline OpsKernel ops_dense_choice(int64_t M, int64_t N, int64_t K, bool gated, int cus)
{
    if (M <= 32) return kOpsRows;
    const int64_t segs = (M + 31) / 32, units = segs * ((N + 15) / 16), tiles = (units + cus - 1) / cus * (gated ? 2 : 1);
    const double rows = 7.0 + (double)tiles * (double)K * (M > 512 ? 0.5e-3 : 0.34e-3) + 3.5 * (double)((tiles - 1) / 8);
    const double mid = ops_mid_cost((double)segs, N, K, gated, cus);
    const double n2 = gated ? 2.0 * (double)N : (double)N;
    const double blocks = (double)((M + 127) / 128) * (double)(((int64_t)n2 + 255) / 256);
    double large;
    if (M > 512) large = std::min(16.0 + 2e-9 * (double)M * n2 * (double)K * (256.0 / cus), ops_gemm_cost((double)((M + 127) / 128), N, K, gated, cus));
    else if (2 * blocks > cus) large = (double)(int64_t)(blocks / cus + 0.999) * (12.0 + (double)K * 10e-3);   // enough blocks: no split
    else large = 14.0 + 0.085 * (double)M + 0.3e-6 * n2 * (double)(K >> 2) * (256.0 / cus);
    if (std::min(rows, mid) >= large) return kOpsGemm;
    return rows <= mid ? kOpsRows : kOpsMid;
}

template <bool kGated>
int run_ops(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, int64_t K, void *workspace,
            int64_t workspace_bytes, hipStream_t s)
{
    const int64_t rows = kGated ? 2 * (int64_t)e.N : e.N;
    const int force = g_ops_kernel.load(std::memory_order_relaxed);
    if (force == kOpsGeneric || !ops_mfma_ok(x, codes, grid, g, rows, K) || !(ops_x_near(g, K) || ops_x_by_block(g, K)))
        return run_ops_generic<kGated>(x, codes, grid, g, e, K, s);
    if (!ops_x_near(g, K)) return run_ops_gemm<kGated>(x, codes, grid, g, e, K, s);
    // The kernels whose loads add the offset of a row inside a tile (of 16 rows of W, of 32 of x) to the tile's take K up to 2^23, as
    // the plain product's do: the sums stay below 2^32.  Longer ones go to the matrix-matrix kernel, whose lanes have one offset.
    const bool k_ok = K <= (1 << 23), rows_ok = k_ok && ops_jobs_fit(g, 4, e.N), mid_ok = k_ok && ops_jobs_fit(g, kMidRows, e.N);
    const int cus = cu_count();
    // One row of a matrix: the batch-1 kernels' bodies
    const bool one_row = force < 0 && k_ok && !g.offsets && g.R == 1 && (K & 255) == 0;
    if (!kGated && one_row && (e.N & 3) == 0 && ((int64_t)e.N + 15) / 16 <= cus && ops_stream_lds(K) <= kLdsMax)
        return launch_ops_stream(x, codes, grid, g, e, K, s);
    if (one_row && !e.out_f32 && ops_share(e.N, kGated) <= 8 && gemv_q8_enabled()) return launch_ops_q8d<kGated>(x, codes, grid, g, e, K, s);
    // 8-bit operands, two rows per segment.  One or two rows of a dense call: from three tiles per compute unit on, or two on a
    // long K, and not on a short one; elsewhere the 16-bit kernel is as fast or faster and its sums are exact products' (graph
    // launches, us, 8-bit / 16-bit, two rows: 1024 -> 4096 4.76 / 3.93, 4096 -> 4096 5.10 / 4.72, 11008 -> 4096 7.10 / 6.73, 28672 -> 4096
    // 13.5 / 12.3, 4096 -> 8192 5.52 / 5.36, 8192 -> 8192 7.05 / 7.10, 4096 -> 2 x 2048 5.58 / 5.40, 1024 -> 32000 7.4 / 6.4, 2048 -> 22016 7.1 /
    // 6.5, 512 -> 128000 21.9 / 19.2; but 2560 -> 16384 6.26 / 6.44, 4096 -> 11008 6.20 / 6.29, 4096 -> 22016 8.46 / 9.24, 8192 -> 28672 14.6 /
    // 16.8, 12288 -> 8192 9.4 / 9.9, 28672 -> 8192 16.4 / 17.2, 4096 -> 2 x 11008 8.72 / 9.35, 8192 -> 2 x 28672 30.5 / 35.5).  By
    // expert where few experts have a row and the codes are many (2 x 11008 x 4096, 8 experts, 1 row 12.7, 16-bit 14.4; 2 rows
    // 18.9 / 21.1; but 4 rows 24.7 / 20.6).
    const bool rows8_ok = k_ok && ops_jobs_fit(g, 2, e.N) && !e.out_f32 && (e.residual != e.y || ops_redo_by_number(g, e.N, cus));
    const int64_t share = ops_share(e.N, kGated);
    const bool rows8_pays = g.offsets ? (g.R <= 2 || 4 * (int64_t)g.R <= g.E) && K >= 4096 &&
                                            std::min<int64_t>(g.R, g.E) * rows * (K >> 2) >= (20LL << 20)
                                      : g.R <= 2 && K > 2048 && (share >= 3 || (share == 2 && K >= 12288));
    if (rows8_ok && (force == kOpsRows8 || (force < 0 && rows8_pays && gemv_q8_enabled())))
        return run_ops_rows8<kGated>(x, codes, grid, g, e, K, s);
    if (rows_ok && force == kOpsRows) return run_ops_rows<kGated>(x, codes, grid, g, e, K, s);
    if (mid_ok && force == kOpsMid) return launch_ops_mid<kGated>(x, codes, grid, g, e, K, s);
    if (g.offsets) {
        // Up to eight rows per expert the few-rows kernel, then the one for tens of rows where every wave has a unit, or the
        // matrix-matrix kernel, by their estimates; half a segment and half a tile of every expert are not full
        // (graph launches, us, few rows / tens / matrix-matrix, rows per expert: 2 x 11008 x 4096, 8 experts 4: 56 / 62 / 88, 8: 75 / 68 /
        // 90, 31: 127 / 92 / 181, 64: 224 / 165 / 221, 128: - / 288 / 367, 256: - / 528 / 533; 4096 x 11008, 16 experts 4: 50 / 63 / 74,
        // 8: 74 / 73 / 141, 31: 114 / 100 / 147, 128: - / 288 / 292, 256: - / 533 / 455; 2 x 1408 x 2048, 64 experts 4: 33 / 37 / 51, 8: 47 /
        // 46 / 66, 31: 93 / 65 / 99, 128: - / 159 / 196, 256: - / 294 / 274; but 4096 x 4096, 8 experts, 8 units per workgroup, 12: 20 / 24)
        const int64_t avg = g.R / g.E, units = (int64_t)g.E * ((avg + 31) / 32) * ((e.N + 15) / 16);
        if (force < 0 && rows_ok && (avg < 8 || (avg <= 64 && units <= 8LL * cus))) return run_ops_rows<kGated>(x, codes, grid, g, e, K, s);
        if (force < 0 && mid_ok && ops_mid_cost((double)g.R / 32 + 0.5 * g.E, e.N, K, kGated, cus) <=
                                       ops_gemm_cost((double)g.R / 128 + 0.5 * g.E, e.N, K, kGated, cus))
            return launch_ops_mid<kGated>(x, codes, grid, g, e, K, s);
        return run_ops_gemm<kGated>(x, codes, grid, g, e, K, s);
    }
    const OpsKernel choice = force < 0 ? ops_dense_choice(g.R, e.N, K, kGated, cus) : kOpsGemm;
    if (choice == kOpsRows && rows_ok) return run_ops_rows<kGated>(x, codes, grid, g, e, K, s);
    if (choice == kOpsMid && mid_ok) return launch_ops_mid<kGated>(x, codes, grid, g, e, K, s);
    if (force != kOpsGemm && workspace && workspace_bytes > 0 && g.R >= kSplitKMinM && (K & 63) == 0 && gemm_reg_ok(g.R, rows, K)) {
        const int splits = splitk_plan(g.R, rows, K, workspace_bytes, cus);
        if (splits >= 2) {
            const int st = launch_gemm_partial(x, codes, grid, (float *)workspace, splits, g.R, rows, K, s);
            if (st != 0) return st;
            const int64_t cells = (int64_t)g.R * ((e.N + 3) / 4);
            return launch<false, true>(ops_splitk_kernel<kGated>, dim3((unsigned)((cells + 255) / 256)), dim3(256), 0, s,
                                       (const float *)workspace, e, g.R, splits);
        }
    }
    return run_ops_gemm<kGated>(x, codes, grid, g, e, K, s);
}

int dispatch_ops(const void *x, const void *codes, const void *grid, const Groups &g, const Epi &e, bool gated, int64_t K,
                 void *workspace, int64_t workspace_bytes, hipStream_t s)
{
    return gated ? run_ops<true>(x, codes, grid, g, e, K, workspace, workspace_bytes, s)
                 : run_ops<false>(x, codes, grid, g, e, K, workspace, workspace_bytes, s);
}

// 0: no split
int64_t ops_workspace_bytes(int64_t M, int64_t N, int64_t K, bool gated)
{
    if (M < kSplitKMinM || N < 1 || K < 64 || (K & 63) || M > 65535LL * 128 || N > INT32_MAX / 2 || K > INT32_MAX) return 0;   // first: no overflow below
    const int64_t rows = gated ? 2 * N : N;
    if (!gemm_reg_ok(M, rows, K)) return 0;
    if (ops_dense_choice(M, N, K, gated, cu_count_or_default()) != kOpsGemm && g_ops_kernel.load(std::memory_order_relaxed) != kOpsSplit) return 0;
    const int splits = splitk_plan(M, rows, K, INT64_MAX, cu_count_or_default());
    return splits >= 2 ? (int64_t)splits * M * rows * 4 : 0;
}

const std::vector<KernelInfo> &ops_kernel_table()
{
    static const std::vector<KernelInfo> t = {
#define DMM_K_OPS(G)                                                                                                     \
    kinfo(ops_gemm_kernel<1, G>, gr_smem_bytes(1), true), kinfo(ops_gemm_kernel<2, G>, gr_smem_bytes(2), true),         \
        kinfo(ops_gemm_kernel<4, G>, gr_smem_bytes(4), true)
        DMM_K_OPS(false), DMM_K_OPS(true),
#undef DMM_K_OPS
#define DMM_K_ROWS_X(NT, G, O)                                                                                                    \
    kinfo(ops_rows_kernel<NT, 2, 2, 16, 1, G, O>, kLdsMax, true), kinfo(ops_rows_kernel<NT, 2, 8, 8, 1, G, O>, kLdsMax, true),    \
        kinfo(ops_rows_kernel<NT, 2, 8, 8, 2, G, O>, kLdsMax, true)
#define DMM_K_ROWS(G, O) DMM_K_ROWS_X(2, G, O), DMM_K_ROWS_X(4, G, O), DMM_K_ROWS_X(8, G, O)
        DMM_K_ROWS(false, false), DMM_K_ROWS(true, false), DMM_K_ROWS(false, true), DMM_K_ROWS(true, true),
#undef DMM_K_ROWS
#undef DMM_K_ROWS_X
        kinfo(ops_rows_kernel<8, 4, 8, 8, 1, true, false>, kLdsMax, true),
#define DMM_K_ROWS_4(G)                                                                                                           \
    kinfo(ops_rows_kernel<2, 2, 4, 16, 1, G, true>, kLdsMax, true), kinfo(ops_rows_kernel<4, 2, 4, 16, 1, G, true>, kLdsMax, true), \
        kinfo(ops_rows_kernel<8, 2, 4, 16, 1, G, true>, kLdsMax, true), kinfo(ops_rows_kernel<8, 2, 4, 16, 1, G, false>, kLdsMax, true)
        DMM_K_ROWS_4(false), DMM_K_ROWS_4(true),
#undef DMM_K_ROWS_4
#define DMM_K_OQ8D(G)                                                                                                             \
    kinfo(ops_q8d_kernel<2, 1, 2, G>, kLdsMax, true), kinfo(ops_q8d_kernel<4, 1, 2, G>, kLdsMax, true),                           \
        kinfo(ops_q8d_kernel<6, 1, 3, G>, kLdsMax, true), kinfo(ops_q8d_kernel<8, 1, 2, G>, kLdsMax, true)
        DMM_K_OQ8D(false), DMM_K_OQ8D(true),
#undef DMM_K_OQ8D
#define DMM_K_ROWS8(G)                                                                                                            \
    kinfo(ops_rows8_kernel<2, 2, G, true>, kLdsMax, true), kinfo(ops_rows8_kernel<4, 2, G, true>, kLdsMax, true),                 \
        kinfo(ops_rows8_kernel<8, 2, G, true>, kLdsMax, true), kinfo(ops_rows8_kernel<4, 2, G, false>, kLdsMax, true),            \
        kinfo(ops_rows8_kernel<8, 2, G, false>, kLdsMax, true)
        DMM_K_ROWS8(false), DMM_K_ROWS8(true),
#undef DMM_K_ROWS8
#define DMM_K_ROUTE(EV, L) kinfo(route_choose_kernel<EV, L, false>, kLdsMax, false), kinfo(route_choose_kernel<EV, L, true>, kLdsMax, false)
        DMM_K_ROUTE(1, 16), DMM_K_ROUTE(2, 16), DMM_K_ROUTE(4, 16), DMM_K_ROUTE(8, 16), DMM_K_ROUTE(16, 16),
        DMM_K_ROUTE(1, 64), DMM_K_ROUTE(2, 64), DMM_K_ROUTE(4, 64), DMM_K_ROUTE(8, 64), DMM_K_ROUTE(16, 64),
#undef DMM_K_ROUTE
        kinfo(route_place_kernel, kLdsMax, false), kinfo(ops_stream_kernel, kLdsMax, true),
        kinfo(ops_mid_kernel<4, false>, kMidBytes, true), kinfo(ops_mid_kernel<4, true>, kMidBytes, true),
    };
    return t;
}

// ------------------------------------------------------------------ choice of experts
// 64 tokens per block; more tokens take more words per expert's mask, so that the second kernel's sums over the
// blocks stay short (512 blocks, up to eight words)
inline int route_words(int64_t T)
{
    int w = 1;
    while (w < 8 && T > (int64_t)w * 64 * 512) w *= 2;
    return w;
}
inline int64_t route_blocks(int64_t T) { return (T + 64 * route_words(T) - 1) / (64 * route_words(T)); }

template <int EV, int L>
int launch_route(const RouteArgs &a, int64_t blocks, hipStream_t s)
{
    const size_t masks = (size_t)a.E * a.words * 8;
    if (blocks == 1)
        return launch(route_choose_kernel<EV, L, true>, dim3(1), dim3(1024), masks + (size_t)(a.E + 1 + 64 * a.k) * 4, s, a);
    const int st = launch<true, false>(route_choose_kernel<EV, L, false>, dim3((unsigned)blocks), dim3(1024), masks, s, a);
    if (st != 0) return st;
    int parts = 0;   // lanes per expert, a power of two up to 64
    while (parts < 6 && (2 << parts) * a.E <= 1024) parts++;
    return launch<false, true>(route_place_kernel, dim3((unsigned)blocks), dim3(1024), masks + (size_t)(2 * a.E + 1) * 4, s, a, (int)blocks,
                               parts);
}

// ------------------------------------------------------------------ the operators on host memory
// Plain loops, the same order of roundings as the device (sums in fp32, one rounding at the store).
inline float host_load(const void *p, int64_t i, int type)
{
    if (type == DMM_F32) return reinterpret_cast<const float *>(p)[i];
    if (type == DMM_BF16) {
        const uint32_t u = (uint32_t)reinterpret_cast<const uint16_t *>(p)[i] << 16;
        return __builtin_bit_cast(float, u);
    }
    return (float)reinterpret_cast<const half_t *>(p)[i];
}

inline void host_store(void *p, int64_t i, int type, float v)
{
    if (type == DMM_F32) reinterpret_cast<float *>(p)[i] = v;
    else reinterpret_cast<half_t *>(p)[i] = (half_t)v;
}

// The two GELUs in 64 bits: in 32, their arguments' roundings would show in the tails.
inline float host_act(float z, int act)
{
    switch (act) {
        case DMM_ACT_RELU: return z < 0.f ? 0.f : z;
        case DMM_ACT_SILU: return z / (1.f + expf(-z));
        case DMM_ACT_GELU: return (float)(0.5 * z * erfc(z * -0.70710678118654752440));
        case DMM_ACT_GELU_TANH: return (float)(z / (1.0 + exp(-1.59576912160573071176 * (z + 0.044715 * z * z * z))));
        default: return z;
    }
}

int host_ops(const void *x, int64_t T, const int32_t *rows, const void *codes, const void *grid, const float *scales, int scale_cols,
             const int32_t *offsets, const dmm_epilogue &ep, void *y, int64_t R, int64_t E, int64_t N, int64_t K)
{
    const int64_t kc = K >> 3, N2 = ep.gated ? 2 * N : N;
    const half_t *xh = (const half_t *)x;
    std::atomic<int> failed{0};
    std::atomic<int> *failed_p = &failed;
    for (int64_t e = 0; e < E; e++) {
        int64_t lo = 0, hi = R;
        if (offsets) {
            lo = offsets[e] < 0 ? 0 : offsets[e] > R ? R : offsets[e];
            hi = offsets[e + 1] < lo ? lo : offsets[e + 1] > R ? R : offsets[e + 1];
        }
        if (lo == hi) continue;
        float s = ep.scale, su = ep.scale_up;
        if (scales) {
            s *= scales[e * scale_cols];
            su *= scales[e * scale_cols + scale_cols - 1];
        }
        const uint16_t *ce = (const uint16_t *)codes + e * N2 * kc;
        host_parallel_rows(N, 2 * K * (hi - lo + 1), [=, &ep](int64_t n0, int64_t n1) {
            half_t *w = (half_t *)malloc((size_t)(2 * K + 1) * sizeof(half_t));   // a decoded row, and its partner
            if (!w) {
                failed_p->store(1, std::memory_order_relaxed);
                return;
            }
            for (int64_t n = n0; n < n1; n++) {
                host_decode_row(ce + n * kc, (const half_t *)grid, kc, w);
                if (ep.gated) host_decode_row(ce + (N + n) * kc, (const half_t *)grid, kc, w + K);
                for (int64_t p = lo; p < hi; p++) {
                    const int64_t t = rows ? rows[p] : p;
                    float v = 0.f, u = 0.f;
                    if (t >= 0 && t < T) {
                        for (int64_t k = 0; k < K; k++) v += (float)xh[t * K + k] * (float)w[k];
                        if (ep.gated)
                            for (int64_t k = 0; k < K; k++) u += (float)xh[t * K + k] * (float)w[K + k];
                    }
                    float z = v * s;
                    if (ep.bias) z += host_load(ep.bias, e * N2 + n, ep.bias_type);
                    z = host_act(z, ep.activation);
                    if (ep.gated) {
                        float zu = u * su;
                        if (ep.bias) zu += host_load(ep.bias, e * N2 + N + n, ep.bias_type);
                        z *= zu;
                    }
                    if (ep.residual) z += host_load(ep.residual, p * N + n, ep.residual_type);
                    host_store(y, p * N + n, ep.out_type, z);
                }
            }
            free(w);
        });
    }
    return failed.load(std::memory_order_relaxed) ? DMM_ERR_HOST_MEMORY : DMM_OK;
}

int check_route(const void *logits, int type, int64_t T, int64_t E, int64_t k, int scoring, const void *weights, const void *experts,
                const void *offsets, const void *rows, const void *slots)
{
    if (T < 0 || E < 1 || k < 1 || k > E) return DMM_ERR_BAD_SHAPE;
    if (type != DMM_F16 && type != DMM_F32 && type != DMM_BF16) return DMM_ERR_BAD_SHAPE;
    if (scoring != DMM_SCORE_SOFTMAX && scoring != DMM_SCORE_SIGMOID) return DMM_ERR_BAD_SHAPE;
    if (E > kRouteMaxE || k > kRouteMaxK || T > kRouteMaxT || T * k > INT32_MAX) return DMM_ERR_TOO_LARGE;
    if (!offsets || (T > 0 && (!logits || !weights || !experts || !rows || !slots))) return DMM_ERR_NULL_POINTER;
    if (!aligned(logits, type_bytes(type)) || !aligned(weights, 4) || !aligned(experts, 4) || !aligned(offsets, 4) || !aligned(rows, 4) ||
        !aligned(slots, 4))
        return DMM_ERR_MISALIGNED;
    return DMM_OK;
}

int check_combine(const void *y, int y_type, const void *slots, const void *weights, const void *residual, int residual_type,
                  const void *out, int out_type, int64_t R, int64_t T, int64_t k, int64_t N)
{
    if (R < 0 || T < 0 || k < 0 || N < 0) return DMM_ERR_BAD_SHAPE;
    if (!type_ok(y_type) || !type_ok(out_type) || (residual && !type_ok(residual_type))) return DMM_ERR_BAD_SHAPE;
    if (T == 0 || N == 0) return DMM_OK;
    if (!out || (k > 0 && (!slots || !weights)) || (k > 0 && R > 0 && !y)) return DMM_ERR_NULL_POINTER;
    if (!aligned(y, type_bytes(y_type)) || !aligned(slots, 4) || !aligned(weights, 4) || !aligned(out, type_bytes(out_type)) ||
        (residual && !aligned(residual, type_bytes(residual_type))))
        return DMM_ERR_MISALIGNED;
    if (R > INT32_MAX || T > INT32_MAX || k > INT32_MAX || N > INT32_MAX - 4096) return DMM_ERR_TOO_LARGE;
    if (!residual_ok(residual, residual_type, out, out_type, T * N)) return DMM_ERR_OVERLAP;
    return DMM_OK;
}
