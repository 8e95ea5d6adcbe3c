// What the two translation units of the library share on the host side: launch plumbing and the
// per-device set-up (defined in dmm_host.h).
// Part of libdmm: included by dmm.hip and dmm_ops.hip inside namespace dmm; not a translation unit of
// its own.

extern thread_local hipEvent_t tls_start;   // dmm_set_kernel_events
extern thread_local hipEvent_t tls_stop;

template <typename T>
struct same_type { typedef T type; };

// Enqueue one kernel; the status is what the launch call itself returns (no look at the
// thread's last-error state, which may hold somebody else's stale error).  kFirst / kLast:
// whether this launch opens / closes the span the timing events bracket (an operator call
// that takes two kernels records start before the first and stop after the second).
template <bool kFirst = true, bool kLast = true, typename... KArgs>
int launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t shmem, hipStream_t stream,
           typename same_type<KArgs>::type... args)
{
    void *argv[] = {(void *)&args...};
    if (tls_start && tls_stop)
        return (int)hipExtLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, argv, shmem, stream,
                                       kFirst ? tls_start : nullptr, kLast ? tls_stop : nullptr, 0);
    return (int)hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, argv, shmem, stream);
}

inline bool aligned(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

constexpr int kLdsMax = 160 * 1024;

// Every kernel that needs more dynamic LDS than the default limit, or whose table addressing
// assumes that its dynamic LDS starts at LDS address 0 (true exactly when the kernel has no
// static LDS, which dmm_init verifies from the function's attributes).
struct KernelInfo {
    const void *fn;
    int dynamic_lds;   // bytes to allow; 0 = default limit is enough
    bool lds_base0;
};

template <typename... KArgs>
KernelInfo kinfo(void (*k)(KArgs...), int lds, bool base0) { return KernelInfo{reinterpret_cast<const void *>(k), lds, base0}; }

// the kernels of dmm_ops.hip, for dmm_init
const std::vector<KernelInfo> &ops_kernel_table();

struct DeviceState;
int ensure_ready(hipStream_t stream, const DeviceState **out = nullptr);   // set-up of the current device on its first call
int cu_count();              // compute units of the current device, after ensure_ready
int cu_count_or_default();   // the same for pure queries: 256 before the device is set up

// the plain product's split of K, which the product with an epilogue shares: the plan, and the kernel that leaves
// fp32 partial sums in part [splits][M][N]
constexpr int kSplitKMinM = 17;   // smallest M that splits (up to M = 16 the matrix-vector kernels are as fast or faster)
int gemm_reg_tm(int64_t M);       // rows of x per block / 32
bool gemm_reg_ok(int64_t M, int64_t N, int64_t K);
int splitk_plan(int64_t M, int64_t N, int64_t K, int64_t workspace_bytes, int cus);
int launch_gemm_partial(const void *x, const void *codes, const void *grid, float *part, int splits, int64_t M, int64_t N, int64_t K,
                        hipStream_t stream);

bool gemv_q8_enabled();   // dmm_set_gemv_8bit: may the library pick kernels on 8-bit operands?
