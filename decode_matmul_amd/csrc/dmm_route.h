// The choice of experts, the lists the grouped product reads, and the weighted sum of the experts' rows.
// Part of libdmm: included by dmm_ops.hip inside namespace dmm; not a translation unit of its own.

// ------------------------------------------------------------------ choice of experts
// L lanes per token: sixteen (four tokens per wave) for up to 256 experts and sixteen choices, else the whole wave.
// Lane l of them holds logits l, L + l, ... of the row as ordered unsigned keys (equal numbers have equal keys, -inf and
// NaN have key 0 and are never chosen); k times the largest key is found with a maximum over the lanes, then the
// lowest index that holds it.  Lane j keeps choice j.  The vector ALU bounds it: sixteen lanes per token take a
// fifth of the instructions per token that a wave per token took.  16384 tokens, 8 of 128 experts: 14.2 us for both kernels, 9 and
// 7 by the trace; 24 tokens, 2 of 16, one launch: 5.1 us a call, 2.8 by the trace.
//
// The lists.  Sorting by expert must keep the order of the tokens, and within a token an expert is chosen
// once, so a row's place is: first row of its expert + number of earlier tokens that chose the expert.  A workgroup
// takes 64 * words tokens and keeps, per expert, a bit mask of the tokens that chose it (set by LDS atomics: the
// order of ors does not matter, so the result does not depend on it); a place inside the block is a population count.
// The masks and their counts go to the workspace and a second kernel adds the counts of the blocks before; with one
// block the same launch does it all.
// Every block of the second kernel reads the counts of all blocks, which sets the limit on the tokens of a call.
constexpr int kRouteMaxE = 1024, kRouteMaxK = 64;
constexpr int64_t kRouteMaxT = 1 << 24;

__device__ __forceinline__ uint32_t route_key(float v)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);   // -0 and 0 are equal
    if (v != v || u == 0xFF800000u) return 0u;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float route_unkey(uint32_t key)
{
    return __builtin_bit_cast(float, (key & 0x80000000u) ? key & 0x7FFFFFFFu : ~key);
}

// reductions over the L lanes of a token, the result in each of them: sixteen lanes by rotations of the row
template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_row(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xF, 0xF, true);
}
struct MaxU32 {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};
struct MinU32 {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a < b ? a : b; }
};
struct OrU32 {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a | b; }
};
struct AddF32 {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const
    {
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
    }
};
template <int L, class Op>
__device__ __forceinline__ uint32_t lanes_reduce(uint32_t v, Op op)
{
    v = op(v, dpp_row<0x128>(v));   // row_ror:8
    v = op(v, dpp_row<0x124>(v));   // row_ror:4
    v = op(v, dpp_row<0x122>(v));   // row_ror:2
    v = op(v, dpp_row<0x121>(v));   // row_ror:1
    if constexpr (L == 64) {
        v = op(v, (uint32_t)__shfl_xor((int)v, 16, kWave));
        v = op(v, (uint32_t)__shfl_xor((int)v, 32, kWave));
    }
    return v;
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v)
{
    return __builtin_bit_cast(float, lanes_reduce<L>(__builtin_bit_cast(uint32_t, v), AddF32()));
}

__device__ __forceinline__ float route_load(const void *p, int64_t i, int type)
{
    if (type == DMM_F32) return reinterpret_cast<const float *>(p)[i];
    const uint16_t b = reinterpret_cast<const uint16_t *>(p)[i];
    if (type == DMM_BF16) return __builtin_bit_cast(float, (uint32_t)b << 16);
    return (float)__builtin_bit_cast(half_t, b);
}

struct RouteArgs {
    const void *logits;
    int type, T, E, k, sigmoid, normalize;
    float *weights;      // [T][k]
    int32_t *experts;    // [T][k]
    int32_t *offsets;    // [E + 1]
    int32_t *rows;       // [T k]
    int32_t *slots;      // [T][k]
    uint64_t *masks;     // workspace: [blocks][E][words]
    int32_t *counts;     // workspace: [E][blocks4]
    int words;           // tokens per block / 64
    int blocks4;         // blocks, rounded up to a multiple of four
};

template <int EV>
struct RouteRow {
    float v[EV];
};
// token t < a.T, or nothing (-inf)
template <int EV, int L>
__device__ __forceinline__ RouteRow<EV> route_row(const RouteArgs &a, int t, bool live, int l)
{
    RouteRow<EV> r;
#pragma unroll
    for (int i = 0; i < EV; i++) {
        const int e = i * L + l;
        r.v[i] = live && e < a.E ? route_load(a.logits, (int64_t)t * a.E + e, a.type) : -__builtin_inff();
    }
    return r;
}

// choice of one token by L lanes, l this lane's number among them; returns this lane's choice (expert or -1, l < k)
template <int EV, int L>
__device__ __forceinline__ int route_token(const RouteArgs &a, const RouteRow<EV> &row, int t, bool live, int l)
{
    const float (&v)[EV] = row.v;
    uint32_t key[EV];
#pragma unroll
    for (int i = 0; i < EV; i++) key[i] = route_key(v[i]);
    int mine = -1;
    float val = 0.f, big = 0.f;
    for (int j = 0; j < a.k; j++) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < EV; i++) best = key[i] > best ? key[i] : best;
        best = lanes_reduce<L>(best, MaxU32());
        uint32_t at = ~0u;   // the lowest index that holds it
#pragma unroll
        for (int i = EV - 1; i >= 0; i--) at = key[i] == best ? (uint32_t)(i * L + l) : at;
        at = lanes_reduce<L>(at, MinU32());
#pragma unroll
        for (int i = 0; i < EV; i++) key[i] = at == (uint32_t)(i * L + l) ? 0u : key[i];
        if (best != 0) {   // else nothing is left to choose, now and in the rounds to come
            const float f = route_unkey(best);
            if (j == 0) big = f;
            if (l == j) {
                mine = (int)at;
                val = f;
            }
        }
    }
    // weights.  softmax: exp(v - largest) over the sum of the chosen ones, or of the whole row; a NaN anywhere in the
    // row shows in all its weights.  sigmoid over the sum of the chosen ones: exp(v) / (1 + exp(v)) = exp(min(v, 0)) /
    // (1 + exp(-|v|)), numerators relative to the largest choice's, so that a row of very low logits does not end in 0 / 0.
    float w, total = 1.f;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < EV; i++) bad |= v[i] != v[i] ? 1u : 0u;
    bad = lanes_reduce<L>(bad, OrU32());
    if (a.sigmoid) {
        if (a.normalize) w = mine >= 0 ? expf(fminf(val, 0.f) - fminf(big, 0.f)) / (1.f + expf(-fabsf(val))) : 0.f;
        else w = mine >= 0 ? epi_sigmoid(val) : 0.f;
    } else {
        w = mine >= 0 ? expf(val - big) : 0.f;
        if (!a.normalize) {
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < EV; i++) part += expf(v[i] - big);   // -inf: 0
            total = lanes_sum<L>(part);
        }
    }
    if (a.normalize) total = lanes_sum<L>(l < a.k ? w : 0.f);
    if (live && l < a.k) {
        w = mine >= 0 ? w / total : 0.f;
        if (bad) w = __builtin_nanf("");
        a.weights[(int64_t)t * a.k + l] = w;
        a.experts[(int64_t)t * a.k + l] = mine;
    }
    return mine;
}

// Kernel 1: weights and experts of the block's tokens, masks and counts per expert.  kOne: the only block (up to 64
// tokens), which writes the lists as well.  A wave has the next token's logits on their way while it chooses for
// one.  LDS: masks [E][words], then (kOne) first rows [E + 1] and the choices.
template <int EV, int L, bool kOne>
__global__ __launch_bounds__(1024) void route_choose_kernel(RouteArgs a)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char route_smem[];
    uint64_t *mask = reinterpret_cast<uint64_t *>(route_smem);
    int *first = reinterpret_cast<int *>(mask + a.E * a.words);
    int *chosen = first + a.E + 1;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int t0 = (int)blockIdx.x * 64 * a.words;
    const int nt = a.T - t0 < 64 * a.words ? a.T - t0 : 64 * a.words;
    constexpr int kPer = 64 / L;   // tokens per wave
    const int l = lane % L, sub = lane / L;
    RouteRow<EV> next = route_row<EV, L>(a, t0 + wave * kPer + sub, wave * kPer + sub < nt, l);
    for (int i = tid; i < a.E * a.words; i += 1024) mask[i] = 0;
    __syncthreads();
    for (int i0 = wave * kPer; i0 < nt; i0 += 16 * kPer) {
        const RouteRow<EV> row = next;
        const int i = i0 + sub;
        if (i0 + 16 * kPer < nt) next = route_row<EV, L>(a, t0 + i + 16 * kPer, i + 16 * kPer < nt, l);
        const int e = route_token<EV, L>(a, row, t0 + i, i < nt, l);
        if (i < nt && l < a.k) {
            if (e >= 0) atomicOr(reinterpret_cast<unsigned long long *>(&mask[e * a.words + (i >> 6)]), 1ull << (i & 63));
            if (kOne) chosen[i * a.k + l] = e;
        }
    }
    __syncthreads();
    if constexpr (!kOne) {
        for (int e = tid; e < a.E; e += 1024) {
            int c = 0;
            for (int w = 0; w < a.words; w++) {
                const uint64_t m = mask[e * a.words + w];
                a.masks[((int64_t)blockIdx.x * a.E + e) * a.words + w] = m;
                c += __builtin_popcountll(m);
            }
            a.counts[(int64_t)e * a.blocks4 + blockIdx.x] = c;
        }
    } else {
        if (wave == 0) {
            int base = 0;
            for (int e0 = 0; e0 < a.E; e0 += 64) {
                const int e = e0 + lane;
                const int c = e < a.E ? __builtin_popcountll(mask[e]) : 0;
                const int s = wave_scan(c, lane);
                if (e < a.E) {
                    first[e] = base + s - c;
                    a.offsets[e] = base + s - c;
                }
                base += __builtin_amdgcn_readlane(s, 63);
            }
            if (lane == 0) {
                first[a.E] = base;
                a.offsets[a.E] = base;
            }
        }
        __syncthreads();
        for (int p = tid; p < nt * a.k; p += 1024) {
            const int t = p / a.k, e = chosen[p];
            int s = -1;
            if (e >= 0) {
                s = first[e] + __builtin_popcountll(mask[e] & ((1ull << t) - 1));
                a.rows[s] = t;
            }
            a.slots[p] = s;
            if (p >= first[a.E]) a.rows[p] = -1;
        }
    }
}

// Kernel 2, one workgroup per block of kernel 1: first rows of every expert from the counts of all blocks, then the
// lists of this block's tokens.  `parts` neighbouring lanes share an expert and read its counts, which lie side by
// side, four at a time; what else the block needs (its masks, its first choices) is on its way meanwhile.
// LDS: masks [E][words], totals [E], first rows of this block [E + 1].
__global__ __launch_bounds__(1024) void route_place_kernel(RouteArgs a, int blocks, int parts_log2)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char route_smem[];
    uint64_t *mask = reinterpret_cast<uint64_t *>(route_smem);
    int *total = reinterpret_cast<int *>(mask + a.E * a.words), *first = total + a.E;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = blockIdx.x;
    const int t0 = b * 64 * a.words;
    const int nt = a.T - t0 < 64 * a.words ? a.T - t0 : 64 * a.words;
    const int32_t *experts = a.experts + (int64_t)t0 * a.k;
    const int mine = tid < nt * a.k ? experts[tid] : -1;
    for (int i = tid; i < a.E * a.words; i += 1024) mask[i] = a.masks[(int64_t)b * a.E * a.words + i];
    const int parts = 1 << parts_log2, part = tid & (parts - 1), e = tid >> parts_log2;
    int tot = 0, bef = 0;   // all blocks, the blocks before this one
    if (e < a.E) {
        typedef int i4_t __attribute__((ext_vector_type(4)));
        const i4_t *src = reinterpret_cast<const i4_t *>(a.counts + (int64_t)e * a.blocks4);
#pragma unroll 4
        for (int i = part; i < a.blocks4 / 4; i += parts) {
            const i4_t c = src[i];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int v = i * 4 + j < blocks ? c[j] : 0;   // the last four: only those that exist
                tot += v;
                bef += i * 4 + j < b ? v : 0;
            }
        }
    }
    for (int off = parts >> 1; off > 0; off >>= 1) {
        tot += __shfl_xor(tot, off, kWave);
        bef += __shfl_xor(bef, off, kWave);
    }
    if (e < a.E && part == 0) {
        total[e] = tot;
        first[e] = bef;
    }
    __syncthreads();
    if (wave == 0) {
        int base = 0;
        for (int e0 = 0; e0 < a.E; e0 += 64) {
            const int ee = e0 + lane;
            const int c = ee < a.E ? total[ee] : 0;
            const int s = wave_scan(c, lane);
            if (ee < a.E) {
                first[ee] += base + s - c;
                if (b == 0) a.offsets[ee] = base + s - c;
            }
            base += __builtin_amdgcn_readlane(s, 63);
        }
        if (lane == 0) {
            first[a.E] = base;
            if (b == 0) a.offsets[a.E] = base;
        }
    }
    __syncthreads();
    for (int i = tid; i < nt * a.k; i += 1024) {
        const int p = t0 * a.k + i, t = i / a.k;
        const int x = i == tid ? mine : experts[i];
        int s = -1;
        if (x >= 0) {
            s = first[x];
            for (int w = 0; w < (t >> 6); w++) s += __builtin_popcountll(mask[x * a.words + w]);
            s += __builtin_popcountll(mask[x * a.words + (t >> 6)] & ((1ull << (t & 63)) - 1));
            a.rows[s] = t0 + t;
        }
        a.slots[p] = s;
        if (p >= first[a.E]) a.rows[p] = -1;   // rows behind the last expert's
    }
}

// ------------------------------------------------------------------ weighted sum of the experts' rows
// out[t] = residual[t] + sum over j, in order, of weights[t][j] * y[slots[t][j]], fp32, one rounding.  Bound by memory: the
// chosen rows are read once, 16 bytes per lane (4099 tokens, 6 rows of 4096 each: 55 us, 4.9 TB/s).  A slot outside y (a choice that was dropped) adds nothing and
// its row is not read.
struct CombineArgs {
    const void *y;
    const int32_t *slots;
    const float *weights;
    const void *residual;
    void *out;
    int y_f32, residual_f32, out_f32;
    int R, T, k, N;
};

// Eight consecutive elements per thread (the last piece of a row: as many as there are).  A row starts wherever t * N puts it:
// global loads and stores of 16 bytes need no more than the element's alignment.
struct __attribute__((packed, aligned(2))) H8Any {
    h8_t v;
};
struct __attribute__((packed, aligned(4))) F4Any {
    f4_t v;
};
struct F8 {
    float v[8];
};

__device__ __forceinline__ F8 combine_load(const void *p, int64_t at, int f32, int n)
{
    F8 r;
    if (n < 8) {
#pragma unroll
        for (int i = 0; i < 8; i++) r.v[i] = i < n ? epi_load(p, at + i, f32) : 0.f;
    } else if (f32) {
        const F4Any *q = reinterpret_cast<const F4Any *>(reinterpret_cast<const float *>(p) + at);
        const f4_t a = q[0].v, b = q[1].v;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            r.v[i] = a[i];
            r.v[4 + i] = b[i];
        }
    } else {
        const h8_t h = reinterpret_cast<const H8Any *>(reinterpret_cast<const half_t *>(p) + at)->v;
#pragma unroll
        for (int i = 0; i < 8; i++) r.v[i] = (float)h[i];
    }
    return r;
}

// kK: rows whose loads are in flight together (the choices of a token go through in groups of kK, in order)
template <int kK>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a)
{
    const int n0 = ((int)blockIdx.x * 256 + (int)threadIdx.x) * 8;
    if (n0 >= a.N) return;
    const int n = a.N - n0 < 8 ? a.N - n0 : 8;
    for (int64_t t = blockIdx.y; t < a.T; t += gridDim.y) {
        F8 acc;
#pragma unroll
        for (int i = 0; i < 8; i++) acc.v[i] = 0.f;
        const int64_t at = t * a.N + n0;
        F8 res = acc;
        if (a.residual) res = combine_load(a.residual, at, a.residual_f32, n);
        for (int j0 = 0; j0 < a.k; j0 += kK) {
            F8 y[kK];
            float w[kK];
#pragma unroll
            for (int j = 0; j < kK; j++) {
                const int s = j0 + j < a.k ? uniform_load(a.slots + t * a.k, j0 + j) : -1;
                const bool live = s >= 0 && s < a.R;
                w[j] = live ? __builtin_bit_cast(float, uniform_load(reinterpret_cast<const int32_t *>(a.weights) + t * a.k, j0 + j)) : 0.f;
                if (live) {
                    y[j] = combine_load(a.y, (int64_t)s * a.N + n0, a.y_f32, n);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) y[j].v[i] = 0.f;
                }
            }
#pragma unroll
            for (int j = 0; j < kK; j++)
#pragma unroll
                for (int i = 0; i < 8; i++) acc.v[i] = __builtin_fmaf(w[j], y[j].v[i], acc.v[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) acc.v[i] += res.v[i];
        if (n < 8) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < n) {
                    if (a.out_f32) reinterpret_cast<float *>(a.out)[at + i] = acc.v[i];
                    else reinterpret_cast<half_t *>(a.out)[at + i] = (half_t)acc.v[i];
                }
        } else if (a.out_f32) {
            F4Any *o = reinterpret_cast<F4Any *>(reinterpret_cast<float *>(a.out) + at);
            o[0].v = f4_t{acc.v[0], acc.v[1], acc.v[2], acc.v[3]};
            o[1].v = f4_t{acc.v[4], acc.v[5], acc.v[6], acc.v[7]};
        } else {
            h8_t h;
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = (half_t)acc.v[i];
            reinterpret_cast<H8Any *>(reinterpret_cast<half_t *>(a.out) + at)->v = h;
        }
    }
}
