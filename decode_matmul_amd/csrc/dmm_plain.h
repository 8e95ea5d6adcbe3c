// The standalone decoder, the catch-all operator kernel and the split-K reduction.
// Part of libdmm: included by dmm.hip inside namespace dmm, in this order; not a
// translation unit of its own.

// ------------------------------------------------------------------ standalone decoder
// Flat: code i -> halves [8i, 8i+8).  kAligned: each thread takes 8 codes with one
// 16-byte load and issues eight 16-byte stores; otherwise one code per thread.
template <bool kAligned>
__global__ __launch_bounds__(256) void decode_kernel(const uint16_t *__restrict__ codes,
                                                     const void *__restrict__ grid,
                                                     uint16_t *__restrict__ W, int64_t n_codes)
{
    __shared__ DecodeTables tab;
    stage_tables<kAligned>(tab, grid, threadIdx.x, 256);
    __syncthreads();
    if (kAligned) {
        // a wave covers 64 consecutive 32-bit words per step: loads are 256 B per wave,
        // stores 2 KiB per wave, both contiguous.
        const int64_t n_words = n_codes >> 1;
        const uint32_t *cw = reinterpret_cast<const uint32_t *>(codes);
        u4_t *out = reinterpret_cast<u4_t *>(W);
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n_words; i += (int64_t)gridDim.x * 256) {
            u4_t w0, w1;
            decode8x2(cw[i], tab, w0, w1);
            out[2 * i] = w0;
            out[2 * i + 1] = w1;
        }
        if ((n_codes & 1) && blockIdx.x == 0 && threadIdx.x == 0)
            out[n_codes - 1] = decode8(codes[n_codes - 1], tab);
    } else {
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n_codes; i += (int64_t)gridDim.x * 256) {
            u4_t w = decode8(codes[i], tab);
            uint16_t *o = W + i * 8;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                o[2 * j] = (uint16_t)(w[j] & 0xFFFFu);
                o[2 * j + 1] = (uint16_t)(w[j] >> 16);
            }
        }
    }
}

// ------------------------------------------------------------------ generic operator path
// One wave per output row n, lanes stride over the row's codes, dot products on the
// vector ALU with fp32 accumulation, DPP/shuffle reduction across the wave.  Handles any
// M, N, K % 8 == 0 and 2-byte alignment; M is processed in chunks of kMC rows of x.
constexpr int kGenericMC = 4;

__global__ __launch_bounds__(256) void generic_kernel(const uint16_t *__restrict__ x,
                                                      const uint16_t *__restrict__ codes,
                                                      const void *__restrict__ grid, float scale,
                                                      uint16_t *__restrict__ y, int64_t M, int64_t N,
                                                      int64_t K)
{
    __shared__ DecodeTables tab;
    stage_tables<false>(tab, grid, threadIdx.x, 256);
    __syncthreads();
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int64_t kc = K >> 3;
    for (int64_t n = (int64_t)blockIdx.x * 4 + wave; n < N; n += (int64_t)gridDim.x * 4) {
        const uint16_t *crow = codes + n * kc;
        for (int64_t m0 = 0; m0 < M; m0 += kGenericMC) {
            float acc[kGenericMC] = {};
            for (int64_t j = lane; j < kc; j += kWave) {
                u4_t w = decode8(crow[j], tab);
                float wf[8];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    h2_t p = as_h2(w[i]);
                    wf[2 * i] = (float)p[0];
                    wf[2 * i + 1] = (float)p[1];
                }
#pragma unroll
                for (int mm = 0; mm < kGenericMC; mm++) {
                    if (m0 + mm < M) {
                        const uint16_t *xr = x + (m0 + mm) * K + j * 8;
#pragma unroll
                        for (int d = 0; d < 8; d++) {
                            half_t xv = __builtin_bit_cast(half_t, xr[d]);
                            acc[mm] = __builtin_fmaf((float)xv, wf[d], acc[mm]);
                        }
                    }
                }
            }
#pragma unroll
            for (int mm = 0; mm < kGenericMC; mm++) {
                float s = wave_sum(acc[mm]);
                if (lane == 0 && m0 + mm < M) {
                    half_t h = (half_t)(s * scale);
                    y[(m0 + mm) * N + n] = __builtin_bit_cast(uint16_t, h);
                }
            }
        }
    }
}

// ------------------------------------------------------------------ split-K reduction
// y = half(scale * sum_z part[z]) over M * N elements; the order of the sum is fixed, so the
// result does not depend on how the blocks were scheduled.
__global__ __launch_bounds__(256) void splitk_reduce_kernel(const float *__restrict__ part, uint16_t *__restrict__ y,
                                                            int64_t mn, int splits, float scale)
{
    const int64_t i4 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i4 >= mn) return;
    if (i4 + 3 < mn && (mn & 3) == 0) {
        f4_t sacc = *reinterpret_cast<const f4_t *>(part + i4);
        for (int z = 1; z < splits; z++) sacc += *reinterpret_cast<const f4_t *>(part + (int64_t)z * mn + i4);
        u2_t v;
        v[0] = (uint32_t)__builtin_bit_cast(uint16_t, (half_t)(sacc[0] * scale)) |
               ((uint32_t)__builtin_bit_cast(uint16_t, (half_t)(sacc[1] * scale)) << 16);
        v[1] = (uint32_t)__builtin_bit_cast(uint16_t, (half_t)(sacc[2] * scale)) |
               ((uint32_t)__builtin_bit_cast(uint16_t, (half_t)(sacc[3] * scale)) << 16);
        *reinterpret_cast<u2_t *>(y + i4) = v;
    } else {
        for (int64_t i = i4; i < mn && i < i4 + 4; i++) {
            float sacc = part[i];
            for (int z = 1; z < splits; z++) sacc += part[(int64_t)z * mn + i];
            y[i] = __builtin_bit_cast(uint16_t, (half_t)(sacc * scale));
        }
    }
}
