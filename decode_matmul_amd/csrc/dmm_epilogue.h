// What happens to a finished sum of the operators with an epilogue: scale, bias, activation (plain or
// gated), residual, one rounding, store.
// Part of libdmm: included by dmm_ops.hip inside namespace dmm; not a translation unit of its own.

// Everything is in fp32 until the one rounding at the store.  z = scale * sum + bias; a plain call
// gives act(z), a gated one act(z of row n) * (z of row N + n); then the residual is added.
struct Epi {
    const void *bias;       // [E][N], gated [E][2 N]; or null
    const void *residual;   // [M][N]; or null.  May be y itself: every element is read by the thread that writes it
    void *y;                // [M][N]
    const float *scales;    // [E][scale_cols] on the device, on top of scale; or null
    float scale, scale_up;  // scale_up: rows N .. 2 N - 1 of a gated call
    int N;
    int act;
    int scale_cols;
    int bias_f32, residual_f32, out_f32;
};

// 1 / (1 + exp(-z)) to about two units in the last place.  exp(-z) = 2^t (1 + ln 2 * r) with t the rounded product
// z * -log2(e) and r what that product lost: without r the relative error would grow with |z|.  An exponential that
// overflows gives 0.
__device__ __forceinline__ float epi_sigmoid(float z)
{
    constexpr float kLog2e = 1.44269502162933349609f, kLog2eLo = 1.92596299112661746887e-8f, kLn2 = 0.693147182464599609375f;
    const float t = z * -kLog2e;
    const float r = __builtin_fmaf(z, -kLog2e, -t) - z * kLog2eLo;
    const float p = __builtin_amdgcn_exp2f(t);
    const float e = __builtin_fabsf(t) < 127.f ? __builtin_fmaf(p, r * kLn2, p) : p;   // no inf * 0, no inf - inf
    return __builtin_amdgcn_rcpf(1.0f + e);
}

// 0.5 z (1 + tanh(u)) = z / (1 + exp(-2 u)), u = sqrt(2 / pi) (z + 0.044715 z^3): 2 u
__device__ __forceinline__ float epi_tanh_arg(float z) { return 1.59576912160573071176f * __builtin_fmaf(0.044715f * z * z, z, z); }

// z Phi(z) = max(z, 0) - a Phi(-a), a = |z|: nothing cancels for z < 0, where 0.5 z (1 + erf(z / sqrt 2)) loses all its digits
// by -6.  Phi(-a) = exp(-a^2 / 2) Q(a); Q, the normal distribution's tail over its density (times 1 / sqrt(2 pi)), falls
// slowly and is t P(t) with t = 1 / (1 + 0.35 a), P of degree 8 fitted for the least relative error over 0 <= a <= 14.5 (3.2e-8).  a^2 is
// split into a rounded square and what that lost, and so is its product with -log2(e) / 2.  About ten half steps of the tail; 5 %
// less time than erff for 2048 x 11008 outputs of K = 4096 (249 -> 236 us).
__device__ __forceinline__ float epi_gelu(float z)
{
    const float a = __builtin_fminf(__builtin_fabsf(z), 40.f);   // far past the smallest float: no inf * 0
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.35f, a, 1.0f));
    float q = -0.0291580297f;
    q = __builtin_fmaf(q, t, 0.144031614f);
    q = __builtin_fmaf(q, t, -0.255840391f);
    q = __builtin_fmaf(q, t, 0.159321249f);
    q = __builtin_fmaf(q, t, -0.023213394f);
    q = __builtin_fmaf(q, t, 0.105552927f);
    q = __builtin_fmaf(q, t, 0.119821183f);
    q = __builtin_fmaf(q, t, 0.139863536f);
    q = __builtin_fmaf(q, t, 0.139621302f) * t;
    constexpr float kHalfLog2e = 0.721347510814666748047f, kHalfLog2eLo = 9.62981495563308734435e-9f, kLn2 = 0.693147182464599609375f;
    const float s = a * a, t2 = s * -kHalfLog2e;
    const float lost = __builtin_fmaf(s, -kHalfLog2e, -t2) - __builtin_fmaf(__builtin_fmaf(a, a, -s), kHalfLog2e, s * kHalfLog2eLo);
    const float p = __builtin_amdgcn_exp2f(t2);
    return (z > 0.f ? z : 0.f * z) - a * q * __builtin_fmaf(p, lost * kLn2, p);   // 0 * z: keeps NaN, and makes one of -inf
}

__device__ __forceinline__ float epi_act(float z, int act)
{
    switch (act) {
        case DMM_ACT_RELU: return z < 0.f ? 0.f : z;   // keeps NaN
        case DMM_ACT_SILU: return z * epi_sigmoid(z);
        case DMM_ACT_GELU: return epi_gelu(z);
        case DMM_ACT_GELU_TANH: return z * epi_sigmoid(epi_tanh_arg(z));
        default: return z;
    }
}

__device__ __forceinline__ float epi_load(const void *p, int64_t i, int f32)
{
    return f32 ? reinterpret_cast<const float *>(p)[i] : (float)reinterpret_cast<const half_t *>(p)[i];
}

// Four elements at a time, wherever a row starts: global loads and stores need no more than the element's alignment.
struct __attribute__((packed, aligned(2))) H4Any {
    h4_t v;
};
struct __attribute__((packed, aligned(4))) F4Row {
    f4_t v;
};

// elements i .. i + 3, zeros from the left-th on
__device__ __forceinline__ f4_t epi_load4(const void *p, int64_t i, int f32, int left)
{
    if (__builtin_expect(left < 4, 0)) {
        f4_t r = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 3; k++)
            if (k < left) r[k] = epi_load(p, i + k, f32);
        return r;
    }
    if (f32) return reinterpret_cast<const F4Row *>(reinterpret_cast<const float *>(p) + i)->v;
    const h4_t h = reinterpret_cast<const H4Any *>(reinterpret_cast<const half_t *>(p) + i)->v;
    return f4_t{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
}

__device__ __forceinline__ void epi_put4(void *p, int64_t i, int f32, int left, f4_t z)
{
    if (__builtin_expect(left < 4, 0)) {
#pragma unroll
        for (int k = 0; k < 3; k++)
            if (k < left) {
                if (f32) reinterpret_cast<float *>(p)[i + k] = z[k];
                else reinterpret_cast<half_t *>(p)[i + k] = (half_t)z[k];
            }
    } else if (f32) {
        reinterpret_cast<F4Row *>(reinterpret_cast<float *>(p) + i)->v = z;
    } else {
        h4_t h;
#pragma unroll
        for (int k = 0; k < 4; k++) h[k] = (half_t)z[k];
        reinterpret_cast<H4Any *>(reinterpret_cast<half_t *>(p) + i)->v = h;
    }
}

struct EpiScale {
    float s, up;
};
__device__ __forceinline__ EpiScale epi_scale(const Epi &e, int expert)
{
    EpiScale r{e.scale, e.scale_up};
    if (__builtin_expect(e.scales != nullptr, 0)) {
        r.s *= e.scales[(int64_t)expert * e.scale_cols];
        r.up *= e.scales[(int64_t)expert * e.scale_cols + e.scale_cols - 1];
    }
    return r;
}

// one output (row, n): v the sum of row n of W, u that of row N + n (gated)
template <bool kGated>
__device__ __forceinline__ void epi_store1(const Epi &e, const EpiScale &sc, float v, float u, int64_t row, int n, int expert)
{
    const int64_t b = (int64_t)expert * (kGated ? 2 * (int64_t)e.N : e.N) + n;
    float z = v * sc.s;
    if (e.bias) z += epi_load(e.bias, b, e.bias_f32);
    z = epi_act(z, e.act);
    if (kGated) {
        float w = u * sc.up;
        if (e.bias) w += epi_load(e.bias, b + e.N, e.bias_f32);
        z *= w;
    }
    const int64_t i = row * e.N + n;
    if (e.residual) z += epi_load(e.residual, i, e.residual_f32);
    if (e.out_f32) reinterpret_cast<float *>(e.y)[i] = z;
    else reinterpret_cast<half_t *>(e.y)[i] = (half_t)z;
}

// The activation of four values side by side, which hides the latency of the exponentials.  kSmall: GELU, by far the
// longest, one value after the other in a loop (the vector turned by one element each time), for kernels that
// have no registers to spare.
template <bool kSmall>
__device__ __forceinline__ f4_t epi_act4(f4_t z, int act)
{
    if (act == DMM_ACT_NONE) return z;
    if (act == DMM_ACT_SILU || act == DMM_ACT_GELU_TANH) {
        f4_t t = z;
        if (act == DMM_ACT_GELU_TANH) {
#pragma unroll
            for (int i = 0; i < 4; i++) t[i] = epi_tanh_arg(z[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) z[i] *= epi_sigmoid(t[i]);
        return z;
    }
    if constexpr (kSmall) {
#pragma unroll 1
        for (int i = 0; i < 4; i++) z = f4_t{z[1], z[2], z[3], epi_act(z[0], act)};
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) z[i] = epi_act(z[i], act);
    }
    return z;
}

// What the epilogue of four outputs (row, n .. n + 3), n < N, reads beside the sums: asked for apart from their use, so that a
// kernel can have the loads of several on their way.  A launch meets its epilogue's code cold, a miss for every line
// that a branch leads to, so the way that calls take is kept short and straight and everything else out of it.
struct EpiOperands {
    f4_t bias, bias_up, residual;
};
template <bool kGated>
__device__ __forceinline__ EpiOperands epi_fetch_bias(const Epi &e, int n, int expert)
{
    EpiOperands o;
    o.bias = o.bias_up = o.residual = f4_t{0.f, 0.f, 0.f, 0.f};
    if (e.bias) {
        const int64_t b = (int64_t)expert * (kGated ? 2 * (int64_t)e.N : e.N) + n;
        o.bias = epi_load4(e.bias, b, e.bias_f32, e.N - n);
        if (kGated) o.bias_up = epi_load4(e.bias, b + e.N, e.bias_f32, e.N - n);
    }
    return o;
}
__device__ __forceinline__ f4_t epi_fetch_residual(const Epi &e, int64_t row, int n)
{
    if (!e.residual) return f4_t{0.f, 0.f, 0.f, 0.f};
    return epi_load4(e.residual, row * e.N + n, e.residual_f32, e.N - n);
}
template <bool kGated>
__device__ __forceinline__ EpiOperands epi_fetch4(const Epi &e, int64_t row, int n, int expert)
{
    EpiOperands o = epi_fetch_bias<kGated>(e, n, expert);
    o.residual = epi_fetch_residual(e, row, n);
    return o;
}

// the four outputs; those past N are left out
template <bool kGated, bool kSmall>
__device__ __forceinline__ void epi_finish4(const Epi &e, const EpiScale &sc, const EpiOperands &o, f4_t v, f4_t u, int64_t row, int n)
{
    f4_t z = epi_act4<kSmall>(v * sc.s + o.bias, e.act);
    if (kGated) z *= u * sc.up + o.bias_up;
    z += o.residual;   // zeros if there is none
    epi_put4(e.y, row * e.N + n, e.out_f32, e.N - n, z);
}

template <bool kGated, bool kSmall>
__device__ __forceinline__ void epi_store4(const Epi &e, const EpiScale &sc, const f4_t &v, const f4_t &u, int64_t row, int n, int expert)
{
    if (n >= e.N) return;
    epi_finish4<kGated, kSmall>(e, sc, epi_fetch4<kGated>(e, row, n, expert), v, u, row, n);
}

// ------------------------------------------------------------------ rows by expert
// offsets[e] .. offsets[e + 1] are expert e's rows of y.  The values come from the device and are not checked
// on the host: they are cut to 0 <= first <= last <= R, so that no list, however broken, leads a kernel out of
// its buffers.  No list: one expert with all R rows.
struct Groups {
    const int32_t *offsets;   // [E + 1] or null
    const int32_t *rows;      // [R]: which row of x a row of y is made from; null: the same
    int E, R, T;              // rows of y, rows of x
};

struct GroupRange {
    int lo, hi;
};
__device__ __forceinline__ GroupRange group_range(const Groups &g, int e)
{
    if (!g.offsets) return GroupRange{0, g.R};
    const int a = g.offsets[e], b = g.offsets[e + 1];
    GroupRange r;
    r.lo = a < 0 ? 0 : a > g.R ? g.R : a;
    r.hi = b < r.lo ? r.lo : b > g.R ? g.R : b;
    return r;
}

// row of x for row p of y, -1 for a row of zeros (an entry of the list that points outside x)
__device__ __forceinline__ int group_row(const Groups &g, int p)
{
    const int t = g.rows ? g.rows[p] : p;
    return t >= 0 && t < g.T ? t : -1;
}

// ------------------------------------------------------------------ catch-all
// One wave per output column (a gated call: per pair of rows of W), lanes stride over the codes, dot products on
// the vector ALU, as the catch-all of the plain product: any K % 8 == 0, any alignment, sizes past 32-bit offsets.
// blockIdx.y: the expert.
template <bool kGated>
__global__ __launch_bounds__(256) void ops_generic_kernel(const uint16_t *__restrict__ x, const uint16_t *__restrict__ codes,
                                                          const void *__restrict__ grid, Groups g, Epi epi, int64_t K)
{
    constexpr int kMC = 4, kH = kGated ? 2 : 1;
    __shared__ DecodeTables tab;
    const int e = blockIdx.y;
    const GroupRange gr = group_range(g, e);
    if (gr.lo == gr.hi) return;
    stage_tables<false>(tab, grid, threadIdx.x, 256);
    __syncthreads();
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int64_t kc = K >> 3, N = epi.N;
    const uint16_t *ce = codes + (int64_t)e * kH * N * kc;
    const EpiScale sc = epi_scale(epi, e);
    for (int64_t n = (int64_t)blockIdx.x * 4 + wave; n < N; n += (int64_t)gridDim.x * 4) {
        for (int p0 = gr.lo; p0 < gr.hi; p0 += kMC) {
            const uint16_t *xr[kMC];
#pragma unroll
            for (int m = 0; m < kMC; m++) {
                const int t = p0 + m < gr.hi ? group_row(g, p0 + m) : -1;
                xr[m] = t >= 0 ? x + (int64_t)t * K : nullptr;
            }
            float acc[kH][kMC] = {};
            for (int64_t j = lane; j < kc; j += kWave) {
#pragma unroll
                for (int h = 0; h < kH; h++) {
                    const u4_t w = decode8(ce[(n + h * N) * kc + j], tab);
#pragma unroll
                    for (int m = 0; m < kMC; m++) {
                        if (!xr[m]) continue;
#pragma unroll
                        for (int d = 0; d < 8; d++)
                            acc[h][m] = __builtin_fmaf((float)__builtin_bit_cast(half_t, xr[m][j * 8 + d]), (float)as_h2(w[d >> 1])[d & 1],
                                                       acc[h][m]);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < kMC; m++) {
                const float v = wave_sum(acc[0][m]);
                const float u = kGated ? wave_sum(acc[kH - 1][m]) : 0.f;
                if (lane == 0 && p0 + m < gr.hi) epi_store1<kGated>(epi, sc, v, u, p0 + m, (int)n, e);
            }
        }
    }
}
