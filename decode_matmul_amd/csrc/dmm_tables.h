// Decode tables in the LDS and the scalar decode of one code.
// Part of libdmm: included by dmm.hip and dmm_ops.hip inside namespace dmm; not a
// translation unit of its own.

// ------------------------------------------------------------------ decode tables in LDS
struct DecodeTables {
    u4_t grid[256];   // row i: 8 halves of grid[i][0..7]
    u4_t sign[128];   // row s: 8 halves, +-1.0, dim d negative iff bit d of (s | parity(s) << 7)
};

__device__ __forceinline__ u4_t sign_row(uint32_t s7)
{
    const uint32_t s8 = s7 | ((__builtin_popcount(s7) & 1u) << 7);
    u4_t r;
#pragma unroll
    for (int i = 0; i < 4; i++)   // +-1.0 = 0x3C00 with the sign bit of dim 2i (low half) / 2i+1 (high half)
        r[i] = 0x3C003C00u | (((s8 >> (2 * i)) & 1u) << 15) | (((s8 >> (2 * i + 1)) & 1u) << 31);
    return r;
}

// Fill the tables with `nthreads` threads (tid in [0, nthreads)).  grid16 tells whether the
// global grid pointer may be read 16 bytes at a time.
template <bool kAligned>
__device__ __forceinline__ void stage_tables(DecodeTables &t, const void *grid, int tid, int nthreads)
{
    for (int i = tid; i < 256; i += nthreads) {
        if (kAligned) {
            t.grid[i] = reinterpret_cast<const u4_t *>(grid)[i];
        } else {
            const uint16_t *g = reinterpret_cast<const uint16_t *>(grid) + i * 8;
            u4_t r;
#pragma unroll
            for (int j = 0; j < 4; j++) r[j] = (uint32_t)g[2 * j] | ((uint32_t)g[2 * j + 1] << 16);
            t.grid[i] = r;
        }
    }
    for (int i = tid; i < 128; i += nthreads) t.sign[i] = sign_row((uint32_t)i);
}

__device__ __forceinline__ h2_t as_h2(uint32_t v) { return __builtin_bit_cast(h2_t, v); }
__device__ __forceinline__ uint32_t as_u32(h2_t v) { return __builtin_bit_cast(uint32_t, v); }

// Decode one code (low 16 bits of c) into 8 halves = 4 packed registers.
__device__ __forceinline__ u4_t decode8(uint32_t c, const DecodeTables &t)
{
    u4_t g = t.grid[c & 0xFFu];
    u4_t s = t.sign[(c >> 8) & 0x7Fu];
    uint32_t db = ((c & 0x8000u) * 0x10001u) | 0x34003400u;   // packed (+-0.25, +-0.25)
    h2_t d = as_h2(db);
    u4_t w;
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = as_u32(__builtin_elementwise_fma(as_h2(g[i]), as_h2(s[i]), d));
    return w;
}

// Two codes packed in one 32-bit word (low half = first code).
__device__ __forceinline__ void decode8x2(uint32_t w, const DecodeTables &t, u4_t &w0, u4_t &w1)
{
    u4_t g0 = t.grid[w & 0xFFu];
    u4_t s0 = t.sign[(w >> 8) & 0x7Fu];
    u4_t g1 = t.grid[(w >> 16) & 0xFFu];
    u4_t s1 = t.sign[(w >> 24) & 0x7Fu];
    uint32_t db = (w & 0x80008000u) | 0x34003400u;            // delta of code 0 | delta of code 1 << 16
    h2_t d0 = as_h2((db & 0xFFFFu) * 0x10001u);
    h2_t d1 = as_h2((db >> 16) * 0x10001u);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        w0[i] = as_u32(__builtin_elementwise_fma(as_h2(g0[i]), as_h2(s0[i]), d0));
        w1[i] = as_u32(__builtin_elementwise_fma(as_h2(g1[i]), as_h2(s1[i]), d1));
    }
}

// Sum over the 64 lanes of a wave, in every lane.
__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    return v;
}
