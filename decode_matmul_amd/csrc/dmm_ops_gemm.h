// Matrix-matrix kernel of the operators with an epilogue (many rows of x), dense and by expert, and the
// reduction of split-K sums with the epilogue.
// Part of libdmm: included by dmm_ops.hip inside namespace dmm; not a translation unit of its own.

// gemm_reg_body (dmm_gemm.h) does the product; this is where its block lies and what becomes of its sums.
//   * Dense: block (x, y) has rows 32 TM x of y.  By expert: blockIdx.x counts the 32 TM row tiles of the experts in
//     order, empty ones left out; every wave finds its expert with one 64-lane scan over the offsets, and a
//     block past the last tile ends before its first barrier.  The grid is sized for the worst case,
//     R / (32 TM) + E tiles, because the host does not know the sizes.
//   * Gated: the two 32-row tiles of a wave are the gate's and the up projection's same 32 rows, so a lane holds both
//     factors of its outputs in the same elements of acc[0] and acc[1].
//   * The sums go through the LDS (the tables and x are not needed any more) as a [row of y][column] fp32 tile with a
//     pitch of 260 floats - 16 lanes of the 16-byte writes, one row each, meet 16 different bank groups - and come
//     back row by row: stores and the reads of the residual cover whole lines (512 bytes of a row per wave
//     and load), and the activation's code exists once, in a loop, not once per accumulator element.
// What bounds it: the matrix unit is busy for half of the cycles, the rest is what one wave per SIMD issues beside it, as in the
// plain kernel.  Gate and up of 4096 -> 11008, 2048 rows 371 us (995 TF/s); the same by 8 experts, 4096 rows 839 us (881 TF/s; every
// expert ends in a tile that is not full).
template <bool kGated>
struct GemmOpsPlace {
    static constexpr bool kRagged = true;
    static constexpr int kPitch = kGrBN + 4;
    static constexpr int kOutN = kGated ? kGrBN / 2 : kGrBN;   // columns of y per block
    int m0, m_end, n0, expert;
    const Groups &g;
    const Epi &epi;
    __device__ __forceinline__ int x_base(int m, int K) const   // no list: from the block's first row on
    {
        const int t = g.rows ? group_row(g, m) : m - m0;
        return t < 0 ? kGrOut : t * K * 2;
    }
    __device__ __forceinline__ int w_row(int i, int wave, int l32) const
    {
        if (!kGated) return n0 + wave * 64 + i * 32 + l32;
        const int n = n0 + wave * 32 + l32;
        return n < epi.N ? i * epi.N + n : -1;
    }
    template <int TM>
    __device__ __forceinline__ void finish(const f16_t (&acc)[kGrTN][TM], int wave, int l32, int kq, int tid, unsigned char *smem) const
    {
        static_assert(32 * TM * kPitch * 4 <= gr_smem_bytes(TM), "the sums go where the tables and x were");
        float *tile = reinterpret_cast<float *>(smem);
        __syncthreads();   // everybody is done with the tables and x
        // D layout of 32x32: element e of lane: row (n) = 8*(e/4) + 4*(lane/32) + e%4, column (m) = lane%32
#pragma unroll
        for (int i = 0; i < kGrTN; i++)
#pragma unroll
            for (int j = 0; j < TM; j++)
#pragma unroll
                for (int e4 = 0; e4 < 4; e4++) {
                    const int c = (kGated ? i * kOutN + wave * 32 : wave * 64 + i * 32) + 8 * e4 + 4 * kq;
                    *reinterpret_cast<f4_t *>(tile + (j * 32 + l32) * kPitch + c) =
                        f4_t{acc[i][j][4 * e4], acc[i][j][4 * e4 + 1], acc[i][j][4 * e4 + 2], acc[i][j][4 * e4 + 3]};
                }
        // a thread has one place in the columns for all its rows: the bias comes once, the residual kAhead rows at a time
        constexpr int kPer = kOutN / 4, kStep = 256 / kPer, kAhead = 4;
        const int c = (tid % kPer) * 4, n = n0 + c;
        const EpiScale sc = epi_scale(epi, expert);
        EpiOperands ops;
        if (n < epi.N) ops = epi_fetch_bias<kGated>(epi, n, expert);
        __syncthreads();
        if (n >= epi.N) return;
        const int rows = m_end - m0 < 32 * TM ? m_end - m0 : 32 * TM;
        for (int r0 = tid / kPer; r0 < rows; r0 += kStep * kAhead) {
            f4_t res[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; j++)
                res[j] = r0 + j * kStep < rows ? epi_fetch_residual(epi, m0 + r0 + j * kStep, n) : f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int j = 0; j < kAhead && r0 + j * kStep < rows; j++) {   // (turned by one each time: the activation's code once)
                const int r = r0 + j * kStep;
                const float *src = tile + r * kPitch + c;
                const f4_t v = *reinterpret_cast<const f4_t *>(src);
                const f4_t u = kGated ? *reinterpret_cast<const f4_t *>(src + kOutN) : f4_t{0.f, 0.f, 0.f, 0.f};
                ops.residual = res[0];
#pragma unroll
                for (int i = 0; i + 1 < kAhead; i++) res[i] = res[i + 1];
                epi_finish4<kGated, false>(epi, sc, ops, v, u, m0 + r, n);
            }
        }
    }
};

// Tile `want` of the experts' row tiles (bm rows each) in order: its expert and first row; false past the last.
// By a whole wave, the same answer in all lanes.
__device__ __forceinline__ bool find_tile(const Groups &g, int bm, int want, int lane, int &expert, int &first, int &end)
{
    int base = 0;
    for (int e0 = 0; e0 < g.E; e0 += 64) {
        const int e = e0 + lane;
        GroupRange r{0, 0};
        if (e < g.E) r = group_range(g, e);
        const int c = (int)(((uint32_t)(r.hi - r.lo) + (uint32_t)bm - 1u) / (uint32_t)bm);
        int s = c;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(s, off, kWave);
            if (lane >= off) s += o;
        }
        const uint64_t here = __builtin_amdgcn_ballot_w64(want < base + s);   // lanes from the tile's expert on
        if (here != 0) {
            const int l = __builtin_ctzll(here);
            expert = e0 + l;
            const int before = base + __builtin_amdgcn_readlane(s - c, l);
            first = __builtin_amdgcn_readlane(r.lo, l) + (want - before) * bm;
            end = __builtin_amdgcn_readlane(r.hi, l);
            return true;
        }
        base += __builtin_amdgcn_readlane(s, 63);
    }
    return false;
}

template <int TM, bool kGated>
__global__ __launch_bounds__(256) void ops_gemm_kernel(const uint16_t *__restrict__ x, const uint16_t *__restrict__ codes,
                                                       const void *__restrict__ grid, Groups g, Epi epi, int K)
{
    int expert = 0, first = (int)blockIdx.x * 32 * TM, end = g.R;
    if (g.offsets && !find_tile(g, 32 * TM, (int)blockIdx.x, (int)threadIdx.x & 63, expert, first, end)) return;
    typedef GemmOpsPlace<kGated> Place;
    const Place p{first, end, (int)blockIdx.y * Place::kOutN, expert, g, epi};
    const int rows = kGated ? 2 * epi.N : epi.N;
    // Without a list the block's rows of x follow each other: 31-bit offsets from its first one, wherever that lies.
    const int64_t x_first = g.rows ? 0 : first, x_bytes = (g.T - x_first) * K * 2;
    gemm_reg_body<TM, false, false>(p, x + x_first * K, x_bytes < INT32_MAX ? x_bytes : INT32_MAX,
                                    codes + (int64_t)expert * rows * (K >> 3), rows, grid, K, 1);
}

// y = epilogue(sum over z of part[z]): part [splits][M][N or 2 N] fp32, added in a fixed order.  One thread per four outputs.
template <bool kGated>
__global__ __launch_bounds__(256) void ops_splitk_kernel(const float *__restrict__ part, Epi epi, int M, int splits)
{
    const int n4 = (epi.N + 3) / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)M * n4) return;
    const int64_t m = i / n4;
    const int n = (int)(i - m * n4) * 4;
    const int64_t row = kGated ? 2 * (int64_t)epi.N : epi.N, plane = (int64_t)M * row;
    const float *src = part + m * row + n;
    f4_t v = f4_t{0.f, 0.f, 0.f, 0.f}, u = v;
    for (int z = 0; z < splits; z++) {
        v += epi_load4(src + z * plane, 0, 1, epi.N - n);
        if (kGated) u += epi_load4(src + z * plane + epi.N, 0, 1, epi.N - n);
    }
    epi_store4<kGated, false>(epi, epi_scale(epi, 0), v, u, m, n, 0);
}
