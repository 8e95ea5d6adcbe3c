// The choice of experts, the lists the grouped product reads, and the weighted sum of the experts' rows.
// Part of libdmm: included by dmm_ops.hip inside namespace dmm; not a translation unit of its own.

// ------------------------------------------------------------------ choice of experts
// One wave per token.  A lane holds logits lane, 64 + lane, ... of the row as ordered unsigned keys (equal numbers have
// equal keys, -inf and NaN have key 0 and are never chosen); k times the largest key of the wave is found with a
// maximum over the lanes, and the lowest index that holds it with one ballot per register, lowest register first.
// Lane j keeps choice j.
//
// The lists.  Sorting by expert must keep the order of the tokens, and within a token an expert is chosen
// once, so a row's place is: first row of its expert + number of earlier tokens that chose the expert.  A workgroup
// takes 64 * words tokens and keeps, per expert, a bit mask of the tokens that chose it (set by LDS atomics: the
// order of ors does not matter, so the result does not depend on it); a place inside the block is a population count.
// The masks and their counts go to the workspace and a second kernel adds the counts of the blocks before; with one
// block the same launch does it all.
constexpr int kRouteMaxE = 1024, kRouteMaxK = 64;

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

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)v, off, kWave);
        v = o > v ? o : v;
    }
    return v;
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
    int32_t *counts;     // workspace: [blocks][E]
    int words;           // tokens per block / 64
};

// choice of one token by one wave; returns this lane's choice (expert or -1, lanes < k)
template <int EV>
__device__ __forceinline__ int route_token(const RouteArgs &a, int t, int lane)
{
    float v[EV];
    uint32_t key[EV];
#pragma unroll
    for (int i = 0; i < EV; i++) {
        const int e = i * 64 + lane;
        v[i] = e < a.E ? route_load(a.logits, (int64_t)t * a.E + e, a.type) : -__builtin_inff();
        key[i] = route_key(v[i]);
    }
    int mine = -1;
    float val = 0.f;
    uint32_t top = 0;
    for (int j = 0; j < a.k; j++) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < EV; i++) best = key[i] > best ? key[i] : best;
        best = (uint32_t)__builtin_amdgcn_readfirstlane((int)wave_max_u32(best));
        if (j == 0) top = best;
        if (best == 0) break;   // nothing left to choose
        bool found = false;
#pragma unroll
        for (int i = 0; i < EV; i++) {
            const uint64_t at = __builtin_amdgcn_ballot_w64(key[i] == best);
            if (!found && at != 0) {
                const int l = __builtin_ctzll(at);
                if (lane == l) key[i] = 0;
                if (lane == j) {
                    mine = i * 64 + l;
                    val = route_unkey(best);
                }
                found = true;
            }
        }
    }
    // weights.  softmax: exp(v - largest) over the sum of the chosen ones, or of the whole row; a NaN anywhere in the
    // row shows in all its weights
    float w, total;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < EV; i++) bad = bad || v[i] != v[i];
    bad = __builtin_amdgcn_ballot_w64(bad) != 0;
    const float big = top == 0 ? 0.f : route_unkey(top);
    if (a.sigmoid) {
        w = mine >= 0 ? epi_sigmoid(val) : 0.f;
        total = 1.f;
    } else {
        w = mine >= 0 ? expf(val - big) : 0.f;
        float part = 0.f;
        if (!a.normalize) {
#pragma unroll
            for (int i = 0; i < EV; i++) part += expf(v[i] - big);   // -inf: 0
            total = wave_sum(part);
        }
    }
    if (a.normalize) total = wave_sum(lane < a.k ? w : 0.f);
    if (lane < a.k) {
        w = mine >= 0 ? w / total : 0.f;
        if (bad) w = __builtin_nanf("");
        a.weights[(int64_t)t * a.k + lane] = w;
        a.experts[(int64_t)t * a.k + lane] = mine;
    }
    return mine;
}

// Kernel 1: weights and experts of the block's tokens, masks and counts per expert.  kOne: the only block, which
// writes the lists as well.  LDS: masks [E][words], then (kOne) first rows [E + 1].
template <int EV, bool kOne>
__global__ __launch_bounds__(1024) void route_choose_kernel(RouteArgs a)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char route_smem[];
    uint64_t *mask = reinterpret_cast<uint64_t *>(route_smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int t0 = (int)blockIdx.x * 64 * a.words;
    const int nt = a.T - t0 < 64 * a.words ? a.T - t0 : 64 * a.words;
    for (int i = tid; i < a.E * a.words; i += 1024) mask[i] = 0;
    __syncthreads();
    for (int i = wave; i < nt; i += 16) {
        const int e = route_token<EV>(a, t0 + i, lane);
        if (lane < a.k && e >= 0)
            atomicOr(reinterpret_cast<unsigned long long *>(&mask[e * a.words + (i >> 6)]), 1ull << (i & 63));
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
            a.counts[(int64_t)blockIdx.x * a.E + e] = c;
        }
    } else {
        int *first = reinterpret_cast<int *>(mask + a.E * a.words);
        if (wave == 0) {
            int base = 0;
            for (int e0 = 0; e0 < a.E; e0 += 64) {
                const int e = e0 + lane;
                const int c = e < a.E ? __builtin_popcountll(mask[e * a.words]) : 0;
                int s = c;
#pragma unroll
                for (int off = 1; off < 64; off <<= 1) {
                    const int o = __shfl_up(s, off, kWave);
                    if (lane >= off) s += o;
                }
                if (e < a.E) {
                    first[e] = base + s - c;
                    a.offsets[e] = base + s - c;
                }
                base += __shfl(s, 63, kWave);
            }
            if (lane == 0) {
                first[a.E] = base;
                a.offsets[a.E] = base;
            }
        }
        __syncthreads();
        for (int p = tid; p < nt * a.k; p += 1024) {
            const int t = p / a.k;
            const int e = a.experts[p];   // written by this block, before the barriers
            int s = -1;
            if (e >= 0) {
                s = first[e] + __builtin_popcountll(mask[e * a.words] & ((1ull << t) - 1));
                a.rows[s] = t;
            }
            a.slots[p] = s;
            if (p >= first[a.E]) a.rows[p] = -1;
        }
    }
}

// Kernel 2, one workgroup per block of kernel 1: first rows of every expert from the counts of all blocks, then the
// lists of this block's tokens.  LDS: totals [E], sums over the blocks before [E], first rows [E + 1].
__global__ __launch_bounds__(1024) void route_place_kernel(RouteArgs a)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char route_smem[];
    int *total = reinterpret_cast<int *>(route_smem), *before = total + a.E, *first = before + a.E;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int blocks = gridDim.x, b = blockIdx.x;
    for (int i = tid; i < 2 * a.E; i += 1024) total[i] = 0;
    __syncthreads();
    // threads (part, expert): integer sums, so the order of the additions does not matter
    const int parts = 1024 / a.E > 0 ? 1024 / a.E : 1;
    const int part = tid / a.E;
    if (part < parts) {
        const int e = tid - part * a.E;
        int tot = 0, bef = 0;
        for (int i = part; i < blocks; i += parts) {
            const int c = a.counts[(int64_t)i * a.E + e];
            tot += c;
            bef += i < b ? c : 0;
        }
        atomicAdd(&total[e], tot);
        atomicAdd(&before[e], bef);
    }
    __syncthreads();
    if (wave == 0) {
        int base = 0;
        for (int e0 = 0; e0 < a.E; e0 += 64) {
            const int e = e0 + lane;
            const int c = e < a.E ? total[e] : 0;
            int s = c;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int o = __shfl_up(s, off, kWave);
                if (lane >= off) s += o;
            }
            if (e < a.E) first[e] = base + s - c;
            base += __shfl(s, 63, kWave);
        }
        if (lane == 0) first[a.E] = base;
    }
    __syncthreads();
    if (b == 0)
        for (int e = tid; e <= a.E; e += 1024) a.offsets[e] = first[e];
    const int t0 = b * 64 * a.words;
    const int nt = a.T - t0 < 64 * a.words ? a.T - t0 : 64 * a.words;
    const uint64_t *mask = a.masks + (int64_t)b * a.E * a.words;
    for (int i = tid; i < nt * a.k; i += 1024) {
        const int p = t0 * a.k + i, t = i / a.k;
        const int e = a.experts[p];
        int s = -1;
        if (e >= 0) {
            s = first[e] + before[e];
            for (int w = 0; w < (t >> 6); w++) s += __builtin_popcountll(mask[e * a.words + w]);
            s += __builtin_popcountll(mask[e * a.words + (t >> 6)] & ((1ull << (t & 63)) - 1));
            a.rows[s] = t0 + t;
        }
        a.slots[p] = s;
        if (p >= first[a.E]) a.rows[p] = -1;   // rows behind the last expert's
    }
}

// ------------------------------------------------------------------ weighted sum of the experts' rows
// out[t] = residual[t] + sum over j, in order, of weights[t][j] * y[slots[t][j]], fp32, one rounding.  Bound by memory: the
// chosen rows are read once, 16 bytes per lane.  A slot outside y (a choice that was dropped) adds nothing and
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

// kVec consecutive elements per thread
template <int kVec>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a)
{
    const int n = ((int)blockIdx.x * 256 + (int)threadIdx.x) * kVec;
    if (n >= a.N) return;
    for (int64_t t = blockIdx.y; t < a.T; t += gridDim.y) {
        float acc[kVec];
#pragma unroll
        for (int i = 0; i < kVec; i++) acc[i] = 0.f;
        for (int j = 0; j < a.k; j++) {
            const int s = a.slots[t * a.k + j];
            if (s < 0 || s >= a.R) continue;
            const float w = a.weights[t * a.k + j];
            const int64_t at = (int64_t)s * a.N + n;
#pragma unroll
            for (int i = 0; i < kVec; i++) acc[i] = __builtin_fmaf(w, epi_load(a.y, at + i, a.y_f32), acc[i]);
        }
        const int64_t at = t * a.N + n;
#pragma unroll
        for (int i = 0; i < kVec; i++) {
            if (a.residual) acc[i] += epi_load(a.residual, at + i, a.residual_f32);
            if (a.out_f32) reinterpret_cast<float *>(a.out)[at + i] = acc[i];
            else reinterpret_cast<half_t *>(a.out)[at + i] = (half_t)acc[i];
        }
    }
}
