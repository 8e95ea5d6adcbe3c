// Tens of rows of x per matrix: the product with an epilogue and the product by expert, every wave on rows of W of its own.
// Part of libdmm: included by dmm_ops.hip inside namespace dmm; not a translation unit of its own.

// Between the kernel for few rows (K split over the waves, sums joined per job) and the matrix-matrix kernel (one
// wave per SIMD, tables built again for every tile of y) lies the range where an expert has some tens of rows.  Segments, units and ranges
// are the few-rows kernel's (32 rows per segment); the work inside a workgroup is cut the other way:
//   * a wave owns up to NT 16-row tiles of W for all of K, so nothing is joined: at the end of a job a lane holds
//     four consecutive outputs of one row of y and runs the epilogue on them, without a barrier;
//   * x goes through the LDS for all waves, 32 rows x 512 k at a time (a chunk, 32 KB, two buffers beside the 96 KB of
//     tables): one barrier per chunk.  A wave loads whole rows, one row's 1 KB per instruction, the row's number the
//     same in all lanes, and asks for the chunk after the next barrier while it multiplies this one.  The 16-byte
//     pieces of row m are exchanged by m % 16: writes and reads meet no bank conflict;
//   * in a step of 256 k the two groups of sixteen rows are 16 B operands in registers, which serve all the wave's tiles: one
//     decode of a code feeds two v_mfma_f32_16x16x32_f16;
//   * codes: one load per tile in flight, asked for a whole step ahead, across chunks and jobs.
// Eight waves, two per SIMD: the packed FMAs of one beside the matrix instructions of the other.
// What bounds it: decoding once per 32 rows.  Two waves per SIMD share its issue: vector ALU 42 %, LDS 38 %, matrix unit 26 % of the
// cycles; gathers a word further ahead (also across tiles) change nothing, and 64 rows per segment (a decode for
// four groups, x a step of 256 k at a time, no registers left to read it ahead) took 20 % longer at 31 rows per expert and as
// long at 128.  2 x 1408 x 2048, 64 experts, 1998 rows 60.3 us (382 TF/s); 2 x 11008 x 4096, 8 experts, 512 rows 165 us (560 TF/s).
// LDS map: tables [0, 96K), x buffers [96K, 160K).
constexpr int kMidW = 8, kMidRows = 32, kMidChunk = 512, kMidXBuf = kMidRows * kMidChunk * 2;
constexpr int kMidBytes = kSTablesBytes + 2 * kMidXBuf;
static_assert(kMidBytes <= 160 * 1024, "tables and two chunks of x have to fit the LDS");

template <int NT, bool kGated>
__global__ __launch_bounds__(64 * kMidW) void ops_mid_kernel(OpsRowsArgs args)
{
    constexpr int W = kMidW, CG = 2;
    constexpr int NU = W * (kGated ? NT / 2 : NT);   // units of a full job: unit u is wave u % W's, its (u / W)-th
    constexpr int kOut = (int)0x80000000;
    static_assert(!kGated || NT % 2 == 0, "gate and up tiles in pairs");
    extern __shared__ __attribute__((aligned(256))) unsigned char smem_raw[];
    const uint16_t *__restrict__ x = args.x;
    const uint16_t *__restrict__ codes = args.codes;
    const Groups g = args.g;
    const int K = args.K, N = args.epi.N;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15;
    const int q = lane >> 4;
    const int n_steps = (K + 255) >> 8;
    const int n_chunks = (n_steps + 1) >> 1;
    const int row_bytes = K >> 2;
    const int w_rows = kGated ? 2 * N : N;
    const int upn = (N + 15) >> 4;
    const uint32_t lane_base = (uint32_t)c16 * 16u;
    const uint32_t quarter_bits = 0x34003400u;

    const u4_t grow = tid < 256 ? reinterpret_cast<const u4_t *>(args.grid)[tid] : u4_t{0u, 0u, 0u, 0u};
    OpsCursor cur{};
    const GroupRange first = ops_first_ranges(g, lane);
    stream_stage_signs<64 * W>(smem_raw, tid);   // needs no load: while the list of the experts' rows is on its way
    __builtin_amdgcn_sched_barrier(0);
    if (!ops_range<kMidRows, NU, NU / 4>(g, first, upn, lane, cur)) return;   // the whole workgroup, before any barrier
    struct Job {
        OpsItem it;
        int row[4];   // byte offsets of this wave's rows of x, 8 i + wave; kOut: none
    };
    auto next_job = [&]() {
        Job j{ops_next_job<kMidRows>(g, cur), {kOut, kOut, kOut, kOut}};
        int t[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int m = j.it.row + 8 * i + wave, mc = m < g.R ? m : g.R - 1;
            t[i] = g.rows ? uniform_load(g.rows, mc) : m;
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (j.it.n > 0 && j.it.row + 8 * i + wave < j.it.row_end && (uint32_t)t[i] < (uint32_t)g.T) j.row[i] = t[i] * K * 2;
        return j;
    };

    const __amdgpu_buffer_rsrc_t xrsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(x), 0, (int)((int64_t)g.T * K * 2), 0x00020000);
    // load i of a chunk: row 8 i + wave, piece `lane`; rows that do not exist and pieces past K are zeros without an access
    u4_t xv[4];
    auto load_x = [&](const Job &j, int chunk) {
        const int xoff = chunk * kMidChunk + lane * 8 < K ? lane * 16 : kOut;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool ok = j.row[i] != kOut;
            xv[i] = __builtin_amdgcn_raw_buffer_load_b128(xrsrc, ok ? xoff : kOut, ok ? j.row[i] + chunk * (kMidChunk * 2) : 0, 0);
        }
    };
    const uint32_t xs = lds_addr(smem_raw) + (uint32_t)kSTablesBytes;
    // row 8 i + wave: 16 bytes of piece `lane` in slot x_slot(lane) ^ (row % 16)
    const uint32_t xs_w0 = xs + (uint32_t)(wave * 1024 + ((x_slot(lane) ^ wave) << 4)), xs_w1 = xs + (uint32_t)(wave * 1024 + ((x_slot(lane) ^ (wave + 8)) << 4));
    auto store_x = [&](int buf) {
#pragma unroll
        for (int i = 0; i < 4; i++) lds_write16(((i & 1) ? xs_w1 : xs_w0) + (uint32_t)(buf * kMidXBuf + i * 8192), xv[i]);
    };
    const uint32_t xs_r = xs + (uint32_t)(c16 * 1024 + ((x_slot(8 * q) ^ c16) << 4));

    const int voff = c16 * row_bytes + q * 16;
    u4_t cw[NT];
    // the code word of tile t for a step (of the job's K); nothing where the tile or the step does not exist
    auto issue = [&](const Job &j, int step, int t) {
        const int u = wave + (kGated ? t >> 1 : t) * W;
        const bool ok = u < j.it.n && step < n_steps;
        const __amdgpu_buffer_rsrc_t crsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t *>(codes) + (int64_t)j.it.expert * w_rows * (K >> 3), 0, w_rows * row_bytes, 0x00020000);
        const int wrow = (j.it.unit + u) * 16 + (kGated ? (t & 1) * N : 0);
        cw[t] = __builtin_amdgcn_raw_buffer_load_b128(crsrc, voff, ok ? wrow * row_bytes + step * 64 : kOut, 0);
    };

    Job job = next_job();
    load_x(job, 0);
#pragma unroll
    for (int t = 0; t < NT; t++) issue(job, 0, t);
    stream_stage_grid<64 * W>(smem_raw, grow, tid);
    store_x(0);
    __syncthreads();

    f4_t acc[NT][CG];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int gi = 0; gi < CG; gi++) acc[t][gi] = f4_t{0.f, 0.f, 0.f, 0.f};

    int buf = 0;
    while (job.it.n > 0) {
        const int mine = (job.it.n - wave + W - 1) / W * (kGated ? 2 : 1);   // this wave's tiles (0 or fewer: none)
        Job nx = job;
        for (int c = 0; c < n_chunks; c++) {
            const bool last = c + 1 == n_chunks;
            if (last) nx = next_job();
            load_x(nx, last ? 0 : c + 1);
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const int step = 2 * c + s;
                u4_t xb[CG][8];
#pragma unroll
                for (int gi = 0; gi < CG; gi++)
#pragma unroll
                    for (int i = 0; i < 8; i++) xb[gi][i] = lds_read16((xs_r ^ (uint32_t)(16 * i)) + (uint32_t)(buf * kMidXBuf + gi * 16384 + s * 512));
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if (t < mine && step < n_steps) fd_tile_step<true, CG>(cw[t], lane_base, quarter_bits, xb, acc[t]);
                    if (s == 0) issue(job, step + 1, t);
                    else issue(nx, last ? 0 : step + 1, t);
                }
            }
            store_x(buf ^ 1);   // last read before the barrier that opened this chunk
            __syncthreads();
            buf ^= 1;
        }
        // D layout of 16x16: lane holds rows 4 q + i of W against column c16, i.e. outputs n = 16 unit + 4 q + i of row c16
        if (mine > 0) {
            const Epi epi = rows_args_copy().epi;
            const EpiScale sc = epi_scale(epi, job.it.expert);
#pragma unroll
            for (int t = 0; t < NT; t += kGated ? 2 : 1) {
                if (t >= mine) break;
                const int n = (job.it.unit + wave + (kGated ? t >> 1 : t) * W) * 16 + 4 * q;
                if (n >= N) continue;
                EpiOperands ops = epi_fetch_bias<kGated>(epi, n, job.it.expert);   // one for both groups of rows
#pragma unroll
                for (int gi = 0; gi < CG; gi++) {
                    const int m = job.it.row + gi * 16 + c16;
                    if (m >= job.it.row_end) continue;
                    ops.residual = epi_fetch_residual(epi, m, n);
                    epi_finish4<kGated, true>(epi, sc, ops, acc[t][gi], acc[kGated ? t + 1 : t][gi], m, n);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int gi = 0; gi < CG; gi++) acc[t][gi] = f4_t{0.f, 0.f, 0.f, 0.f};
        job = nx;
    }
}
