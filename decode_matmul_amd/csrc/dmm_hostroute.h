// Decoding and row loops on host memory.
// Part of libdmm: included by dmm.hip and dmm_ops.hip inside namespace dmm; not a translation unit of
// its own.

// ------------------------------------------------------------------ the operator on host memory
// The reference's own CPU path is a scalar decode and a triple loop (/root/reference/test_decode_matmul.py:29-71);
// this is the same thing for the half-precision form, in plain C++ for tensors that live in host
// memory: no GPU is involved and no GPU call is made.  Not a fallback: device pointers never come
// here, the entry points below are separate ones.  One rounding per weight (the fp32 sum of a half
// and +-1/4 is exact), fp32 sums over k in ascending order, rows of W spread over host threads.
inline void host_decode_row(const uint16_t *codes, const half_t *grid, int64_t kc, half_t *w)
{
    for (int64_t j = 0; j < kc; j++) {
        const uint32_t c = codes[j];
        const uint32_t idx = c & 0xFFu, s7 = (c >> 8) & 0x7Fu;
        const uint32_t s8 = s7 | ((uint32_t)(__builtin_popcount(s7) & 1) << 7);
        const float shift = (c & 0x8000u) ? -0.25f : 0.25f;
        for (int d = 0; d < 8; d++) {
            const float g = (float)grid[idx * 8 + d];
            w[j * 8 + d] = (half_t)(((s8 >> d) & 1u ? -g : g) + shift);
        }
    }
}

// Rows [0, n_rows) split over host threads; body(n0, n1) must not throw.  Threads cost about 50 us
// each to start, so only work of 2^24 multiply-adds or more (several milliseconds on one core) gets
// any, and never more than one per 2^22.  If a thread cannot be started the rows it was to
// take run on the calling thread.
template <typename F>
void host_parallel_rows(int64_t n_rows, int64_t work_per_row, F body) noexcept
{
    const int64_t work = n_rows * work_per_row;
    unsigned threads = std::thread::hardware_concurrency();
    if (threads == 0) threads = 1;
    if (threads > 16) threads = 16;
    if ((int64_t)threads > (work >> 22)) threads = (unsigned)(work >> 22);
    if ((int64_t)threads > n_rows) threads = (unsigned)n_rows;
    if (work < (1 << 24) || threads < 2) {
        body(0, n_rows);
        return;
    }
    std::thread pool[16];
    unsigned started = 0;
    for (unsigned t = 1; t < threads; t++) {
        try {
            pool[started] = std::thread([=] { body(n_rows * t / threads, n_rows * (t + 1) / threads); });
        } catch (...) {   // std::system_error: no more threads to be had
            body(n_rows * t / threads, n_rows);
            break;
        }
        started++;
    }
    body(0, n_rows / threads);
    for (unsigned t = 0; t < started; t++) pool[t].join();
}
