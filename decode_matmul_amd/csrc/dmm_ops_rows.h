// Few rows of x per matrix: the product with an epilogue and the product by expert on 16-bit operands.
// Part of libdmm: included by dmm_ops.hip inside namespace dmm; not a translation unit of its own.

// ------------------------------------------------------------------ the work, cut into jobs
// A segment is up to SR rows of y of one expert (a dense call is one expert); a unit is a segment times 16 columns of
// y: one 16-row tile of W, or for a gated call two, the gate's and the up projection's.  Every segment is cut into the same
// number of jobs, whose sizes differ by at most one unit, and the jobs of all segments are dealt out as contiguous ranges
// that differ by at most one job, one range per workgroup and one workgroup per compute unit, whatever the experts'
// sizes are: an expert with many rows simply has more segments, and the workgroups that walk its other segments at the
// same time find its codes in the caches.  The number of jobs per segment is the one that a cost of kFixed units per job
// and one per unit favours: as many as r rounds of jobs have room for, for the best of four r.
//
// A job is what gemv_f16d_kernel does: chunk of k steps outside, one step per wave; the slice of x of the step
// through the wave's own piece of LDS into eight B operands; tiles inside, every tile's accumulator in registers; code
// loads in a ring of D per wave, which here runs on into the next job (and so do the loads of x).  At the end of a
// job the partial sums go through the pieces, a thread adds up four outputs over the waves in order and runs the
// epilogue on them.
// What bounds it: decoding, on the vector ALU (half of the cycles) and the LDS (45 %; four gathers of 16 bytes per two codes, no bank
// conflicts), beside 18 % on the matrix unit: 11008 -> 4096 by 16 experts, 48 rows on 15 of them 56.0 us, 169 MB of codes at
// 3.0 TB/s; one matrix and few rows: a launch, a pass of the tables and one or two steps per wave (13 rows, 4096 -> 11007, GELU,
// 7.3 us).
// LDS map: tables [0, 96K), then W pieces of XI KB.
struct OpsCursor {
    int expert, row, row_end;   // segment: rows row .. of an expert whose rows end at row_end
    int part, left;             // next job inside the segment, jobs left in the range
    int parts, base, extra;     // jobs per segment; units per job, one more for the first `extra` of them
};

typedef __attribute__((address_space(4))) const int32_t const_i32_t;

// an element of a list that no kernel writes meanwhile, at the same place in all lanes: through the scalar cache
__device__ __forceinline__ int uniform_load(const int32_t *p, int i)
{
    return __builtin_amdgcn_readfirstlane(reinterpret_cast<const_i32_t *>(reinterpret_cast<uintptr_t>(p))[i]);
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ GroupRange uniform_range(const Groups &g, int e)
{
    const int a = uniform_load(g.offsets, e), b = uniform_load(g.offsets, e + 1);
    GroupRange r;
    r.lo = a < 0 ? 0 : a > g.R ? g.R : a;
    r.hi = b < r.lo ? r.lo : b > g.R ? g.R : b;
    return r;
}

// inclusive sum over the lanes of a wave
__device__ __forceinline__ int wave_scan(int v, int lane)
{
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(v, off, kWave);
        if (lane >= off) v += o;
    }
    return v;
}

__device__ __forceinline__ int cut_up(const GroupRange &r, int by) { return (int)(((uint32_t)(r.hi - r.lo) + (uint32_t)by - 1u) / (uint32_t)by); }

// the first 64 experts' rows, one per lane: asked for at a kernel's start, ahead of work that needs no list
__device__ __forceinline__ GroupRange ops_first_ranges(const Groups &g, int lane)
{
    GroupRange first{0, 0};
    if (g.offsets && lane < g.E) first = group_range(g, lane);
    return first;
}

// Where 16-byte piece p of a step of x lies in its row (before the exchange by the row's number): pieces 8 .. 15 behind 16 .. 23.
// A 16-byte LDS read is served sixteen lanes at a time, half of them of one quarter of the wave and half of the next; the
// two read pieces 8 apart, which must not differ in the bank then.
__device__ __forceinline__ int x_slot(int p) { return (p & ~24) | (p >> 1 & 8) | (p << 1 & 16); }

// the workgroup's range of jobs; false: it has none
template <int SR, int NU, int kFixed>
__device__ __forceinline__ bool ops_range(const Groups &g, const GroupRange &first, int upn, int lane, OpsCursor &c)
{
    int segs, first_scan = 0;
    if (!g.offsets) {
        segs = (g.R + SR - 1) / SR;
    } else {
        first_scan = wave_scan(cut_up(first, SR), lane);
        segs = __builtin_amdgcn_readlane(first_scan, 63);
        for (int e0 = 64; e0 < g.E; e0 += 64) {
            GroupRange r{0, 0};
            if (e0 + lane < g.E) r = group_range(g, e0 + lane);
            segs += __builtin_amdgcn_readlane(wave_scan(cut_up(r, SR), lane), 63);
        }
    }
    if (segs == 0) return false;
    const uint32_t wgs = gridDim.x, least = ((uint32_t)upn + NU - 1u) / NU;   // fewest jobs a segment can be cut into
    uint32_t parts = least;
    {
        // (the quotients by reciprocals: one too few or too many costs balance, nothing else)
        const float inv = __builtin_amdgcn_rcpf((float)segs) * (float)wgs;
        uint32_t r = (uint32_t)((float)least * __builtin_amdgcn_rcpf(inv) + 0.999f);
        r = r < 1u ? 1u : r;
        float best = 3e38f;
#pragma unroll
        for (int i = 0; i < 4; i++, r++) {
            uint32_t p = (uint32_t)((float)r * inv + 0.001f);
            p = p > (uint32_t)upn ? (uint32_t)upn : p < least ? least : p;
            const float rounds = (float)(uint32_t)((float)p * __builtin_amdgcn_rcpf(inv) + 0.999f);
            const float cost = rounds * ((float)kFixed + (float)(uint32_t)((float)upn * __builtin_amdgcn_rcpf((float)p) + 0.999f));
            if (cost < best * 0.999f) {
                best = cost;
                parts = p;
            }
        }
    }
    parts = (uint32_t)uniform((int)parts);
    const uint32_t jobs = (uint32_t)segs * parts;   // below 2^31 (ops_jobs_fit)
    const uint32_t b = blockIdx.x, q = jobs / wgs, rest = jobs - q * wgs;
    const uint32_t j0 = b * q + (b < rest ? b : rest);
    c.left = (int)(q + (b < rest ? 1u : 0u));
    if (c.left == 0) return false;
    const int seg = (int)(j0 / parts);
    c.part = (int)(j0 - (uint32_t)seg * parts);
    c.parts = (int)parts;
    c.base = (int)((uint32_t)upn / parts);
    c.extra = upn - c.base * (int)parts;
    if (!g.offsets) {
        c.expert = 0;
        c.row = seg * SR;
        c.row_end = g.R;
    } else {
        int base = 0;
        for (int e0 = 0;; e0 += 64) {   // seg < segs: found
            GroupRange r = first;
            int s = first_scan;
            if (e0 > 0) {
                r = GroupRange{0, 0};
                if (e0 + lane < g.E) r = group_range(g, e0 + lane);
                s = wave_scan(cut_up(r, SR), lane);
            }
            const uint64_t here = __builtin_amdgcn_ballot_w64(seg < base + s);
            if (here != 0 || e0 + 64 >= g.E) {
                const int l = here != 0 ? __builtin_ctzll(here) : 0;
                const int before = base + __builtin_amdgcn_readlane(s - cut_up(r, SR), l);
                c.expert = e0 + l;
                c.row = __builtin_amdgcn_readlane(r.lo, l) + (seg - before) * SR;
                c.row_end = __builtin_amdgcn_readlane(r.hi, l);
                break;
            }
            base += __builtin_amdgcn_readlane(s, 63);
        }
    }
    c = OpsCursor{uniform(c.expert), uniform(c.row), uniform(c.row_end), uniform(c.part), uniform(c.left), uniform(c.parts),
                  uniform(c.base), uniform(c.extra)};
    return true;
}

// a job, and (few-rows kernel) its share of a chunk; n == 0: nothing
struct OpsItem {
    int expert, row, row_end, unit, n, chunk;
};

// the next job of the range
template <int SR>
__device__ __forceinline__ OpsItem ops_next_job(const Groups &g, OpsCursor &c)
{
    OpsItem it{c.expert, c.row, c.row_end, 0, 0, 0};
    if (c.left == 0) return it;
    it.n = c.base + (c.part < c.extra ? 1 : 0);
    it.unit = c.part * c.base + (c.part < c.extra ? c.part : c.extra);
    it.row_end = c.row + SR < c.row_end ? c.row + SR : c.row_end;
    c.left--;
    if (++c.part == c.parts && c.left > 0) {   // on to the next segment
        c.part = 0;
        c.row += SR;
        if (c.row >= c.row_end && g.offsets) {
            GroupRange r{0, 0};
            while (r.lo == r.hi && c.expert + 1 < g.E) r = uniform_range(g, ++c.expert);
            c.row = r.lo;
            c.row_end = r.hi;
        }
    }
    return it;
}

// The kernel's one argument, so that its address in the constant kernel-argument segment is known.  What is needed
// once per job (the epilogue) is read from there when it is needed, not held in scalar registers through the loop.
struct OpsRowsArgs {
    const uint16_t *x, *codes;
    const void *grid;
    Groups g;
    Epi epi;
    int K;
    int units_q, units_r;   // dense calls of one segment: units per workgroup, one more for the first units_r
};
typedef __attribute__((address_space(4))) const OpsRowsArgs const_rows_args_t;

__device__ __forceinline__ const_rows_args_t *rows_args_late()
{
    uint64_t p = (uint64_t)(uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));   // a value of its own: loads through it stay where they are written
    return reinterpret_cast<const_rows_args_t *>((uintptr_t)p);
}

__device__ __forceinline__ OpsRowsArgs rows_args_copy()
{
    OpsRowsArgs a;
    __builtin_memcpy(&a, rows_args_late(), sizeof(a));
    return a;
}

// ---- 8-bit operands (gemv_q8d_kernel's arithmetic) for segments of up to two rows.  The sixteen columns of the
// matrix unit hold four terms of each row (column 4 m + t is term t of row m, of weight 8^-t), the means of the shift
// term ride in columns 4 m and 4 m + 1.  A wave splits the 256 k of its own step into terms - a lane has one piece
// of eight, lanes 32 .. 63 those of the second row - and leaves them in its own piece of LDS: term row 4 m + t at a
// pitch of 272 bytes, the means behind them at a pitch of 80; no barrier, no roles.  What does not fit is found, not
// computed, and left to the 16-bit body in the same launch, with the same jobs: all of them if the grid does not fit
// fp8 (known before the first), and those that met an x that is not finite (the terms of an infinity mean
// nothing), which store nothing here.
// What bounds it: the vector ALU, two thirds of the cycles (gate and up of 8192 -> 28672, one row, 30.2 us, 3.9 TB/s of codes; of 4096 ->
// 11008 by two of eight experts, one row each, 17.8 us, 2.5 TB/s).
constexpr int kO8TermPitch = 272, kO8MeanPitch = 80;
constexpr int kO8Means = 8 * kO8TermPitch;
constexpr int kO8Piece = kO8Means + 4 * kO8MeanPitch + 64;   // 2560
constexpr int kO8Flags = kSTablesBytes + 16 * kO8Piece;      // 16 votes, 2 words for jobs that are not finite, 64 zero bytes
constexpr int kO8Bytes = kO8Flags + 128 + 64;
static_assert(kO8Bytes <= 160 * 1024, "tables and pieces have to fit the LDS");

// XI, W, CG as in gemv_f16d_kernel: 2 XI rows of x per group, W waves, CG groups of sixteen rows per segment; SR: rows of
// a segment, CG * 2 XI or fewer.
// kOne: a dense call of one segment whose workgroups have one job each (up to NU units): the range comes from the
// host, rows of x follow each other, and the loop has only chunks to count (11008 -> 4096 with one row: 8.1 us as a
// job of the general form, 6.8 like this).
// kQ8: 8-bit operands, XI = 1.
// todo: the jobs to do, one bit each, the last bit for all from there on (kSome; otherwise all).  Returns the jobs left to do.
template <int NT, int D, int XI, int W, int CG, bool kGated, bool kOne, int SR, bool kQ8, bool kSome>
__device__ __forceinline__ uint32_t ops_rows_body(const OpsRowsArgs &args, uint32_t todo)
{
    const uint16_t *__restrict__ x = args.x;
    const uint16_t *__restrict__ codes = args.codes;
    const Groups g = args.g;
    const int K = args.K, N = args.epi.N;
    constexpr int CM = 2 * XI;
    constexpr int kPiece = kQ8 ? kO8Piece : XI * 1024;
    constexpr int NU = kGated ? NT / 2 : NT;
    constexpr int kSumUnroll = kOne ? 8 : 4;   // a job with others behind it has their loads in registers: fewer sums side by side
    static_assert(kQ8 ? W == 16 && XI == 1 && CG == 1 : (W == 16 && (XI == 2 || XI == 4)) || (W == 8 && XI == 8), "up to two, four, eight or sixteen rows of x");
    static_assert(CG == 1 || (CG == 2 && XI == 8), "a second group of rows only beside a full first one");
    static_assert(SR <= CG * CM, "the rows of a segment are columns of the product");
    static_assert(kQ8 || fd_lds_bytes(XI, W) <= 160 * 1024, "tables and pieces have to fit the LDS");
    static_assert(NT % D == 0 && (!kGated || NT % 2 == 0), "the ring has to divide the tiles");
    static_assert(NT * 4 * CM * 16 <= kPiece, "the partial sums of a job go through the wave's piece");
    constexpr bool kAhead = W == 8 ? !(NT == 8 && CG == 2) : NT < (XI == 4 && kGated ? 4 : 8);   // a code word's gathers ahead of the word before it, where registers are left
    extern __shared__ __attribute__((aligned(256))) unsigned char smem_raw[];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15;
    const int q = lane >> 4;
    const int n_steps = (K + 255) >> 8;
    const int n_chunks = (n_steps + W - 1) / W;
    const int row_bytes = K >> 2;
    const int w_rows = kGated ? 2 * N : N;
    const int upn = (N + 15) >> 4;
    const uint32_t lane_base = kQ8 ? (uint32_t)(lane & 31) * 8u : (uint32_t)c16 * 16u;
    const uint32_t quarter_bits = 0x34003400u;
    constexpr int kOut = (int)0x80000000;

    const u4_t grow = tid < 256 ? reinterpret_cast<const u4_t *>(args.grid)[tid] : u4_t{0u, 0u, 0u, 0u};
    // the sign rows need no load: written while the list of the experts' rows is on its way
    auto stage_signs = [&]() {
        if constexpr (kQ8) {
            if (tid >= 256 && tid < 512) {
                const int t = tid - 256, row = t >> 1;
                const u2_t sb = sign_bytes((uint32_t)row);
                const uint32_t sg = lds_addr(smem_raw) + (uint32_t)((row * 16 + (t & 1) * 8 + (row & 7)) * 16);
#pragma unroll
                for (int i = 0; i < 8; i++) lds_write16(sg ^ (uint32_t)(i * 16), u4_t{sb[0], sb[1], sb[0], sb[1]});
            }
        } else {
            stream_stage_signs<64 * W>(smem_raw, tid);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    OpsCursor cur{};
    OpsItem it;
    if constexpr (kOne) {
        const int b = (int)blockIdx.x;
        it = OpsItem{0, 0, g.R, b * args.units_q + (b < args.units_r ? b : args.units_r), args.units_q + (b < args.units_r ? 1 : 0), 0};
    } else {
        const GroupRange first = ops_first_ranges(g, lane);
        stage_signs();
        if (!ops_range<SR, NU, 4>(g, first, upn, lane, cur)) return 0u;   // the whole workgroup, before any barrier
        it = ops_next_job<SR>(g, cur);
    }
    // Rows of x: lane l (and l + 32) of row_list holds the list's entry for row l of a job's segment.  The entries are asked
    // for a whole job ahead, so that nobody waits for them behind the codes.
    auto row_list = [&](const OpsItem &j) {
        int m = j.row + (lane & 31);
        if (g.rows) m = g.rows[m < g.R ? m : g.R - 1];
        return m;
    };
    OpsItem nj{};       // the job after this one
    int r_it = 0, r_nj = 0;
    if constexpr (!kOne) {
        r_it = row_list(it);
        nj = ops_next_job<SR>(g, cur);
        r_nj = row_list(nj);
    }

    const __amdgpu_buffer_rsrc_t xrsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(x), 0, (int)((int64_t)g.T * K * 2), 0x00020000);
    u4_t xv[CG][XI];
    // load i of a slice is piece lane % 32 (16 bytes) of row 2 i + lane / 32; rows that do not exist and pieces past K
    // are zeros without a memory access
    auto load_x = [&](const OpsItem &it, int rl, int gi) {
        const int step = it.chunk * W + wave;
        const bool ok = it.n > 0 && step < n_steps;
        const int piece = (int)threadIdx.x & 31;
        const bool inside = ok && step * 256 + piece * 8 < K;
        if constexpr (kOne) {   // rows past the last lie past the end of the buffer
            const int b = inside ? ((((int)threadIdx.x >> 5) & 1) * K + piece * 8) * 2 : kOut;
#pragma unroll
            for (int i = 0; i < XI; i++)
                xv[gi][i] = __builtin_amdgcn_raw_buffer_load_b128(xrsrc, b, ok ? step * 512 + (gi * CM + 2 * i) * 2 * K : kOut, 0);
        } else {
            // byte offset of the lane's row, beyond the buffer where there is none
            const int off = it.row + (lane & 31) < it.row_end && (uint32_t)rl < (uint32_t)g.T ? rl * K * 2 : kOut;
#pragma unroll
            for (int i = 0; i < XI; i++) {
                const int b0 = __builtin_amdgcn_readlane(off, gi * CM + 2 * i), b1 = __builtin_amdgcn_readlane(off, gi * CM + 2 * i + 1);
                const int b = ((int)threadIdx.x & 32) ? b1 : b0;
                xv[gi][i] = __builtin_amdgcn_raw_buffer_load_b128(xrsrc, inside && b != kOut ? b + piece * 16 : kOut, ok ? step * 512 : 0, 0);
            }
        }
    };
    // the wave's piece: row m at a pitch of 512 bytes, its pieces exchanged by m
    const uint32_t piece = lds_addr(smem_raw) + (uint32_t)(kSTablesBytes + wave * kPiece);
    auto xs_w = [&]() { return piece + (uint32_t)((lane >> 5) * 512 + ((x_slot(lane & 31) ^ (lane >> 5)) << 4)); };
    const int xr_row = c16 & (CM - 1);
    const uint32_t xs_r = piece + (uint32_t)(xr_row * 512 + ((x_slot(8 * q) ^ xr_row) << 4));

    const int voff = c16 * row_bytes + q * 16;
    auto issue = [&](u4_t &cwd, const OpsItem &it, int t) {
        const int step = it.chunk * W + wave;
        const bool ok = t < (kGated ? 2 * it.n : it.n) && step < n_steps;
        const __amdgpu_buffer_rsrc_t crsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t *>(codes) + (int64_t)it.expert * w_rows * (K >> 3), 0, w_rows * row_bytes, 0x00020000);
        const int wrow = kGated ? (it.unit + (t >> 1)) * 16 + (t & 1) * N : (it.unit + t) * 16;
        cwd = __builtin_amdgcn_raw_buffer_load_b128(crsrc, voff, ok ? wrow * row_bytes + step * 64 : kOut, 0);
    };

#pragma unroll
    for (int gi = 0; gi < CG; gi++) load_x(it, r_it, gi);
    u4_t cw[D];
    issue(cw[0], it, 0);   // the rest of the ring after the prologue's work, as in gemv_f16d_kernel
    uint32_t *flags = reinterpret_cast<uint32_t *>(smem_raw + kO8Flags);   // kQ8 only
    if constexpr (kOne) stage_signs();
    if constexpr (kQ8) {
        bool exact = true;
        if (tid < 256) {
            const u2_t g8 = grid_row_fp8(grow, exact);
            const uint32_t gg = lds_addr(smem_raw) + (uint32_t)(kSSignBytes + (tid * 16 + (tid & 15)) * 16);   // slot i ^ (tid % 16)
#pragma unroll
            for (int i = 0; i < 16; i++) lds_write16(gg ^ (uint32_t)(i * 16), u4_t{g8[0], g8[1], g8[0], g8[1]});
        } else if (tid >= 512 && tid < 528) {
            flags[16 + tid - 512] = 0u;   // the two words, and what lies up to the zeros
        } else if (tid >= 528 && tid < 544) {
            flags[32 + tid - 528] = 0u;   // the zero bytes the idle columns read
        }
        const bool bad = __builtin_amdgcn_ballot_w64(!exact) != 0;
        if (lane == 0) flags[wave] = bad ? 1u : 0u;
    } else {
        stream_stage_grid<64 * W>(smem_raw, grow, tid);
    }
    // kQ8: the slice of x that has arrived into terms and means, in the wave's piece: for the first item beside the other
    // waves' tables, for the others behind the tiles of the item before
    bool finite = true;   // the x of this wave's steps of the job, so far
    auto split_x = [&]() {
        u2_t tm[4];
        uint32_t mean;
        finite = finite & qd_split_piece(xv[0][0], tm, mean);
        const uint32_t m = (uint32_t)lane >> 5, pc = (uint32_t)lane & 31;
        typedef __attribute__((address_space(3))) u2_t lds_u2_rw_t;
        typedef __attribute__((address_space(3))) uint16_t lds_u16_rw_t;
#pragma unroll
        for (int t = 0; t < 4; t++) *reinterpret_cast<lds_u2_rw_t *>(piece + (m * 4 + t) * kO8TermPitch + pc * 8) = tm[t];
        *reinterpret_cast<lds_u16_rw_t *>(piece + kO8Means + m * 2 * kO8MeanPitch + pc * 2) = (uint16_t)mean;
        *reinterpret_cast<lds_u16_rw_t *>(piece + kO8Means + (m * 2 + 1) * kO8MeanPitch + pc * 2) = (uint16_t)(mean >> 16);
    };
    if constexpr (kQ8) split_x();
#pragma unroll
    for (int d = 1; d < D; d++) issue(cw[d], it, d);
    __syncthreads();
    if constexpr (kQ8) {
        if (__builtin_amdgcn_ballot_w64(flags[lane & 15] != 0) != 0) {
            __syncthreads();   // everybody has read the votes: the other body may have the LDS
            return ~0u;
        }
    }
    // kQ8: this lane's column of the two B operands and of the means inside the piece; idle columns read the zeros
    const uint32_t zeros = lds_addr(smem_raw) + (uint32_t)(kO8Flags + 128);
    const uint32_t o8_t = c16 < 8 ? piece + (uint32_t)(c16 * kO8TermPitch + q * 64) : zeros;
    const uint32_t o8_m = c16 < 8 && (c16 & 3) < 2 ? piece + (uint32_t)(kO8Means + ((c16 >> 2) * 2 + (c16 & 1)) * kO8MeanPitch + q * 16) : zeros;

    f4_t acc[NT][CG];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int gi = 0; gi < CG; gi++) acc[t][gi] = f4_t{0.f, 0.f, 0.f, 0.f};
    int job = 0;
    uint32_t left = 0;   // kQ8: jobs that met an x that is not finite

    while (kOne ? it.chunk < n_chunks : it.n > 0) {
        // (a value of its own every time round: what depends on it is not kept in scalar registers through the loop)
        asm volatile("" : "+s"(it.n), "+s"(it.unit));
        const bool last = it.chunk + 1 == n_chunks;
        OpsItem nx = it;
        nx.chunk++;
        int r_nx = r_it;
        if (!kOne && last) {
            nx = nj;
            r_nx = r_nj;
        }
        const bool step_ok = it.chunk * W + wave < n_steps;
        const int nt = kGated ? 2 * it.n : it.n;
        u4_t xb[CG][kQ8 ? 1 : 8];
        i8_t xb0{}, xb1{};
        h8_t xm{};
        if constexpr (kQ8) {
            const u4_t r0 = lds_read16(o8_t), r1 = lds_read16(o8_t + 16), r2 = lds_read16(o8_t + 32), r3 = lds_read16(o8_t + 48);
            xm = __builtin_bit_cast(h8_t, lds_read16(o8_m));
            xb0 = i8_t{(int)r0[0], (int)r0[1], (int)r0[2], (int)r0[3], (int)r1[0], (int)r1[1], (int)r1[2], (int)r1[3]};
            xb1 = i8_t{(int)r2[0], (int)r2[1], (int)r2[2], (int)r2[3], (int)r3[0], (int)r3[1], (int)r3[2], (int)r3[3]};
            load_x(nx, r_nx, 0);
        } else {
#pragma unroll
            for (int gi = 0; gi < CG; gi++) {
#pragma unroll
                for (int i = 0; i < XI; i++) lds_write16((xs_w() ^ (uint32_t)(32 * i)) + (uint32_t)(1024 * i), xv[gi][i]);
#pragma unroll
                for (int i = 0; i < 8; i++) xb[gi][i] = lds_read16(xs_r ^ (uint32_t)(16 * i));
                load_x(nx, r_nx, gi);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (step_ok && t < nt) {
                if constexpr (kQ8) qd_tile_step(cw[t % D], lane_base, xb0, xb1, xm, acc[t][0]);
                else fd_tile_step<kAhead, CG>(cw[t % D], lane_base, quarter_bits, xb, acc[t]);
            }
            if (t + D < NT) issue(cw[t % D], it, t + D);
            else issue(cw[t % D], nx, t + D - NT);
        }
        if (last) {
            // the end of a job: cell (tile, quarter, column) of every wave's piece, a group of rows at a time
            Epi epi = args.epi;
            if constexpr (!kOne) epi = rows_args_copy().epi;
            // (the thread's number as a value of its own: addresses made from it are not held through the loop)
            int jtid = tid;
            asm volatile("" : "+v"(jtid));
            const int jl = jtid & 63, jc = jl & 15, jq = jl >> 4;
            const EpiScale sc = epi_scale(epi, it.expert);
#pragma unroll
            for (int gi = 0; gi < CG; gi++) {
                if (gi > 0) __syncthreads();   // the readers of the group before are done with the pieces
                // Sixteen waves: the sixteen lanes of a row add one cell up, a wave's sums each (cell c of wave w lies in slot
                // c ^ w, so that they meet no bank conflict), and lane 15 has it; the first cell's operands are asked for ahead of the
                // barrier.  Eight waves of sixteen rows have a cell for every thread: each adds its own up.
                constexpr bool kLanes = W == 16;
                const int n_cells = it.n * 4 * CM;
                auto cell_row = [&](int cell) { return it.row + gi * CM + cell % CM; };
                auto cell_col = [&](int cell) { return (it.unit + cell / (4 * CM)) * 16 + 4 * (cell % (4 * CM) / CM); };
                auto cell_live = [&](int cell) { return cell < n_cells && cell_row(cell) < it.row_end && cell_col(cell) < N; };
                const int cell0 = kLanes ? jtid >> 4 : jtid;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if (t < nt) {
                        f4_t v = acc[t][gi];
                        int col = jc;
                        if constexpr (kQ8) {   // the four terms of a row, with their weights 8^-t, into the lane of column 4 m
                            const float wt = __builtin_bit_cast(float, 0x3F800000u - (((uint32_t)jc & 3u) * 3u << 23));
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                v[e] *= wt;
                                v[e] = dpp_shl_add<1>(v[e], v[e]);
                                v[e] = dpp_shl_add<2>(v[e], v[e]);
                            }
                            col = (jc & 3) == 0 ? jc >> 2 : CM;
                        }
                        if (col < CM)
                            lds_write16(piece + (uint32_t)(((t * 4 + jq) * CM + col) ^ (kLanes ? wave : 0)) * 16, __builtin_bit_cast(u4_t, v));
                    }
                    acc[t][gi] = f4_t{0.f, 0.f, 0.f, 0.f};
                }
                if constexpr (kQ8) {
                    if (__builtin_amdgcn_ballot_w64(!finite) != 0 && jl == 0) flags[16 + (job & 1)] = 1u;
                    finite = true;
                }
                EpiOperands ops0{};
                if (kLanes && jc == 15 && cell_live(cell0)) ops0 = epi_fetch4<kGated>(epi, cell_row(cell0), cell_col(cell0), it.expert);
                __syncthreads();
                bool store = true;
                if constexpr (kQ8) {
                    if (__builtin_amdgcn_ballot_w64(flags[16 + (job & 1)] != 0) != 0) {
                        left |= 1u << (job < 31 ? job : 31);
                        store = false;
                    }
                    if (jtid == 0) flags[17 - (job & 1)] = 0u;   // read by all before this job's barrier, set again behind the next one
                }
                if constexpr (kSome) store = (todo >> (job < 31 ? job : 31) & 1u) != 0;
                const uint32_t sums = lds_addr(smem_raw) + (uint32_t)kSTablesBytes;
                auto slot_of = [&](int cell) { return kGated ? cell / (4 * CM) * 8 * CM + cell % (4 * CM) : cell; };
                if constexpr (kLanes) {
                    for (int c0 = 0; store && c0 < n_cells; c0 += 64) {
                        const int cell = c0 + cell0, slot = slot_of(cell);
                        const uint32_t src = sums + (uint32_t)(jc * kPiece);
                        f4_t v = __builtin_bit_cast(f4_t, lds_read16(src + (uint32_t)((slot ^ jc) << 4))), up = f4_t{0.f, 0.f, 0.f, 0.f};
                        if constexpr (kGated) up = __builtin_bit_cast(f4_t, lds_read16(src + (uint32_t)(((slot + 4 * CM) ^ jc) << 4)));
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            v[e] = row_sum16(v[e]);
                            if (kGated) up[e] = row_sum16(up[e]);
                        }
                        if (jc == 15 && cell_live(cell)) {
                            if (c0 > 0) ops0 = epi_fetch4<kGated>(epi, cell_row(cell), cell_col(cell), it.expert);
                            epi_finish4<kGated, true>(epi, sc, ops0, v, up, cell_row(cell), cell_col(cell));
                        }
                    }
                } else {
                    for (int cell = jtid; store && cell < n_cells; cell += 64 * W) {
                        if (!cell_live(cell)) continue;
                        const uint32_t src = sums + (uint32_t)(slot_of(cell) * 16);
                        f4_t v = f4_t{0.f, 0.f, 0.f, 0.f}, up = v;
#pragma unroll kSumUnroll
                        for (int w = 0; w < W; w++) v += __builtin_bit_cast(f4_t, lds_read16(src + w * kPiece));
                        if constexpr (kGated) {
#pragma unroll kSumUnroll
                            for (int w = 0; w < W; w++) up += __builtin_bit_cast(f4_t, lds_read16(src + 4 * CM * 16 + w * kPiece));
                        }
                        epi_store4<kGated, false>(epi, sc, v, up, cell_row(cell), cell_col(cell), it.expert);
                    }
                }
            }
            job++;
            if constexpr (!kOne) __syncthreads();   // the pieces take the x of the next job next
        }
        if constexpr (kQ8) {
            if (!kOne || nx.chunk < n_chunks) split_x();
        }
        if (!kOne && last) {
            r_it = r_nj;
            nj = ops_next_job<SR>(g, cur);
            r_nj = row_list(nj);
        }
        it = nx;
    }
    if constexpr (kQ8) {
        if (left != 0) __syncthreads();   // the other body may have the LDS
    }
    return left;
}

template <int NT, int D, int XI, int W, int CG, bool kGated, bool kOne>
__global__ __launch_bounds__(64 * W) void ops_rows_kernel(OpsRowsArgs args)
{
    ops_rows_body<NT, D, XI, W, CG, kGated, kOne, 2 * XI * CG, false, false>(args, ~0u);
}

template <int NT, int D, bool kGated, bool kOne>
__global__ __launch_bounds__(1024) void ops_rows8_kernel(OpsRowsArgs args)
{
    const uint32_t left = ops_rows_body<NT, D, 1, 16, 1, kGated, kOne, 2, true, false>(args, ~0u);
    if (left == 0) return;
    const OpsRowsArgs again = rows_args_copy();   // not held in registers meanwhile
    ops_rows_body<NT, D, 2, 16, 1, kGated, kOne, 2, false, true>(again, left);
}

// One row of x on at most one 16-row tile per compute unit, not gated: the streaming kernel's body, whose ring runs two k
// steps ahead where a job of the kernels above has one code load in flight (11008 -> 4096: 6.4 us there, 5.6 here).
__global__ __launch_bounds__(1024) void ops_stream_kernel(OpsRowsArgs args)
{
    const Epi &epi = args.epi;
    const EpiScale sc = epi_scale(epi, 0);
    auto store = [&](int m, int n, const f4_t &v) { epi_store4<false, true>(epi, sc, v, v, m, n, 0); };
    gemv_stream_body_to<1, 16, 2, false, 4>(args.x, args.codes, args.grid, store, 1, epi.N, args.K, args.units_q, args.units_r);
}

// One row of x, up to eight tiles per compute unit: the batch-1 kernel's body on 8-bit operands.  Its roles (tables and the
// split of x in different waves) leave the tables sooner than the jobs' kernel, where every wave splits its own x
// (graph launches, us: 4096 -> 11008 5.1 / 6.2).  What it cannot do goes to the 16-bit body.
template <int NT, bool kGated>
struct Q8dOps {
    static constexpr bool kPairs = kGated;
    const OpsRowsArgs &args;
    __device__ __forceinline__ void store(int n, const f4_t &v) const { store(n, v, v); }
    __device__ __forceinline__ void store(int n, const f4_t &v, const f4_t &u) const
    {
        epi_store4<kGated, true>(args.epi, epi_scale(args.epi, 0), v, u, 0, n, 0);
    }
    __device__ __forceinline__ void hand_over() const
    {
        const OpsRowsArgs again = rows_args_copy();
        ops_rows_body<NT, 2, 2, 16, 1, kGated, true, 4, false, false>(again, ~0u);
    }
};

template <int NT, int U, int D, bool kGated>
__global__ __launch_bounds__(1024) void ops_q8d_kernel(OpsRowsArgs args)
{
    const Q8dOps<NT, kGated> p{args};
    gemv_q8d_body<NT, U, D, false>(p, args.x, args.codes, args.grid, args.epi.N, args.K, args.units_q, args.units_r);
}
