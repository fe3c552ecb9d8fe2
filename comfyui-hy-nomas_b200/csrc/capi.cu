// capi.cu - the extern "C" entry points declared in include/hynomas_b200.h.
//
// Each entry validates its arguments on the host (shapes, null pointers, enum values, the 16-byte
// alignment the vector/TMA paths rely on), checks once per device that it is a compute capability 10.0
// part, launches on the caller's stream and returns an hn_status. Errors never abort the process; the
// message is kept per calling thread for hn_last_error().
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <atomic>
#include <mutex>
#include <string>
#include <utility>

#include <cmath>
#include <cuda.h>
#include <cudaTypedefs.h>

#include "../../include/hynomas_b200.h"
#include "hn_common.cuh"
#include "hn_kernels.h"

namespace hn {

static thread_local std::string t_last_error;

static int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
static int fail(int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    t_last_error = buf;
    return code;
}

static int cuda_fail(cudaError_t e, const char *what) {
    return fail(HN_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
}

constexpr int MAX_DEV = HN_MAX_DEV;
static int g_sms[MAX_DEV];
static int g_arch_ok[MAX_DEV];  // 0 unknown, 1 ok, -1 not sm_100
static std::mutex g_mu;

static int current_device(int *dev) {
    cudaError_t e = cudaGetDevice(dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
    if (*dev < 0 || *dev >= MAX_DEV) return fail(HN_ERR_ARG, "device index %d out of range", *dev);
    return HN_OK;
}

static int check_arch() {
    int dev;
    int rc = current_device(&dev);
    if (rc) return rc;
    if (g_arch_ok[dev] == 0) {
        std::lock_guard<std::mutex> lk(g_mu);
        int major = 0, minor = 0, sms = 0;
        cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
        cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        g_sms[dev] = sms;
        g_arch_ok[dev] = (major == 10 && minor == 0) ? 1 : -1;
        if (g_arch_ok[dev] < 0) t_last_error = "";
    }
    if (g_arch_ok[dev] < 0) {
        int major = 0, minor = 0;
        cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
        cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
        return fail(HN_ERR_ARCH, "device %d is sm_%d%d; this library runs on sm_100a (B200) only", dev, major, minor);
    }
    return HN_OK;
}

static std::atomic<int> g_gemm_sm_reserve{0};
int gemm_sm_reserve() { return g_gemm_sm_reserve.load(std::memory_order_relaxed); }

// stream -> error-word slot (slot 0: the NULL stream, and every stream once the table is full)
static cudaStream_t g_slot_stream[HN_ERR_SLOTS];
static int g_slots_used = 1;

int err_slot(cudaStream_t st) {
    if (st == nullptr) return 0;
    std::lock_guard<std::mutex> lk(g_mu);
    for (int i = 1; i < g_slots_used; ++i)
        if (g_slot_stream[i] == st) return i;
    if (g_slots_used == HN_ERR_SLOTS) return 0;
    g_slot_stream[g_slots_used] = st;
    return g_slots_used++;
}

int num_sms() {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEV) return 148;
    if (g_sms[dev] == 0) {
        int sms = 0;
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        g_sms[dev] = sms > 0 ? sms : 148;
    }
    return g_sms[dev];
}

static inline bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static inline bool al8(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; }
static inline int dsize(int dt) { return dt == HN_DTYPE_FP32 || dt == HN_DTYPE_INT32 ? 4 : 2; }

// A [rows, groups] scale tensor addressed as s[r * rs + g * gs] must not alias two entries: one stride
// must cover the whole extent of the other dimension (row-major: rs >= groups * gs; group-major:
// gs >= rows * rs).
static bool scale_strides_ok(int64_t rows, int64_t groups, int64_t rs, int64_t gs) {
    if (rows <= 1 && groups <= 1) return true;
    if (rows <= 1) return gs >= 1;
    if (groups <= 1) return rs >= 1;
    if (rs < 1 || gs < 1) return false;
    return rs >= groups * gs || gs >= rows * rs;
}

// The device that owns `stream` made current for the duration of an entry point (the caller's current device
// is put back on exit), so a launch, the SM count and the architecture check all refer to the stream's
// device whichever device the calling thread had current. The NULL stream keeps the current device, and so does a
// stream that is being captured into a graph, which may not be asked for its device (a launch from another
// device is then refused by the check of the data's device, or by CUDA).
struct StreamDevice {
    int prev = -1;
    cudaError_t err = cudaSuccess;
    explicit StreamDevice(void *stream) {
        if (stream == nullptr) return;
        int want = 0, cur = 0;
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        err = cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capture);
        if (err != cudaSuccess || capture != cudaStreamCaptureStatusNone) return;
        err = cudaStreamGetDevice(static_cast<cudaStream_t>(stream), &want);
        if (err != cudaSuccess) return;
        err = cudaGetDevice(&cur);
        if (err != cudaSuccess || cur == want) return;
        err = cudaSetDevice(want);
        if (err == cudaSuccess) prev = cur;
    }
    ~StreamDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
    StreamDevice(const StreamDevice &) = delete;
    StreamDevice &operator=(const StreamDevice &) = delete;
};

// The data must live on the launch device: the library enables no peer access, and a kernel handed another
// device's (or host) memory would fault. Checked on each call's main input before anything is launched.
static int check_pointer_device(const void *p, const char *what) {
    cudaPointerAttributes at;
    cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(HN_ERR_ARG, "%s: %p is not memory CUDA knows (%s)", what, p, cudaGetErrorString(e));
    }
    int dev = -1;
    e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
    if (at.type == cudaMemoryTypeManaged) return HN_OK;
    if (at.type != cudaMemoryTypeDevice)
        return fail(HN_ERR_ARG, "%s: %p is not device memory", what, p);
    if (at.device != dev)
        return fail(HN_ERR_ARG, "%s: the data is on device %d but the launch device is %d (pass a stream of the "
                    "data's device, or make that device current for the NULL stream)", what, at.device, dev);
    return HN_OK;
}

static int launched(cudaError_t e, const char *what) {
    if (e != cudaSuccess) return cuda_fail(e, what);
    t_last_error.clear();
    return HN_OK;
}

} // namespace hn

using namespace hn;

// the stream's device made current for the rest of the entry point, then the architecture check on it, and
// the check that the main input `ptr` lives on it
#define CHECK_DEVICE(ptr)                                                                   \
    StreamDevice _stream_device(stream);                                                    \
    if (_stream_device.err != cudaSuccess) return cuda_fail(_stream_device.err, "cudaStreamGetDevice"); \
    do {                                                                                    \
        int _rc = check_arch();                                                             \
        if (_rc == HN_OK) _rc = check_pointer_device((ptr), __func__);                      \
        if (_rc != HN_OK) return _rc;                                                       \
    } while (0)
#define CHECK_ARCH()                                                                        \
    StreamDevice _stream_device(stream);                                                    \
    if (_stream_device.err != cudaSuccess) return cuda_fail(_stream_device.err, "cudaStreamGetDevice"); \
    do {                                                                                    \
        int _rc = check_arch();                                                             \
        if (_rc != HN_OK) return _rc;                                                       \
    } while (0)
#define REQUIRE(cond, code, ...)                      \
    do {                                              \
        if (!(cond)) return fail((code), __VA_ARGS__); \
    } while (0)

extern "C" {

const char *hn_last_error(void) { return t_last_error.c_str(); }

int hn_abi_version(void) { return HN_ABI_VERSION; }

int hn_set_gemm_sm_reserve(int n) {
    if (n < 0 || n > 64) return fail(HN_ERR_ARG, "hn_set_gemm_sm_reserve: n must be in [0, 64]");
    hn::g_gemm_sm_reserve.store(n, std::memory_order_relaxed);
    return HN_OK;
}

int hn_get_gemm_sm_reserve(void) { return hn::gemm_sm_reserve(); }

int hn_num_sms(void) {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
        cudaGetLastError();
        return 0;
    }
    return num_sms();
}

int hn_device_error(void *stream, int *code_host) {
    REQUIRE(code_host != nullptr, HN_ERR_ARG, "code_host is NULL");
    StreamDevice sd(stream);
    if (sd.err != cudaSuccess) return cuda_fail(sd.err, "cudaStreamGetDevice");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return cuda_fail(e, "cudaStreamSynchronize");
    int v = 0;
    e = read_and_clear_device_error(err_slot(st), &v);
    if (e != cudaSuccess) return cuda_fail(e, "reading the device error word");
    *code_host = v;
    if (v & HN_DEVERR_TIMEOUT) return fail(HN_ERR_TIMEOUT, "a device-side wait ran past its limit");
    t_last_error.clear();
    return HN_OK;
}

int hn_selftest_wait_timeout(uint32_t timeout_us, void *stream) {
    CHECK_ARCH();
    REQUIRE(timeout_us > 0 && timeout_us <= 2000000u, HN_ERR_ARG, "timeout_us must be in (0, 2e6]");
    return launched(launch_wait_selftest(timeout_us, static_cast<cudaStream_t>(stream)), "wait self-test launch");
}

int hn_quant_act(const void *x, int64_t ldx, int x_dtype, int64_t M, int64_t K, int kind, int flags, void *q,
                 int64_t ldq, float *s, int64_t s_rs, int64_t s_gs, void *stream) {
    REQUIRE(x && q && s, HN_ERR_ARG, "hn_quant_act: null pointer");
    REQUIRE((flags & ~(HN_QUANT_PER_ROW | HN_QUANT_ROUND_HALF_EVEN)) == 0, HN_ERR_ARG, "hn_quant_act: unknown flags %d", flags);
    REQUIRE(!(flags & HN_QUANT_ROUND_HALF_EVEN) || kind == HN_KIND_INT8, HN_ERR_ARG,
            "hn_quant_act: round-half-even applies to int8 codes (e4m3 always rounds to nearest even)");
    const bool per_row = (flags & HN_QUANT_PER_ROW) != 0;
    REQUIRE(x_dtype == HN_DTYPE_BF16 || x_dtype == HN_DTYPE_FP16 || x_dtype == HN_DTYPE_FP32, HN_ERR_ARG,
            "hn_quant_act: x_dtype %d not bf16/fp16/fp32", x_dtype);
    REQUIRE(kind == HN_KIND_INT8 || kind == HN_KIND_FP8E4M3, HN_ERR_ARG, "hn_quant_act: unknown kind %d", kind);
    REQUIRE(M >= 0 && K > 0 && K % 128 == 0, HN_ERR_SHAPE, "hn_quant_act: need K %% 128 == 0 (M=%lld K=%lld)",
            (long long)M, (long long)K);
    REQUIRE(ldx >= K && ldq >= K, HN_ERR_SHAPE, "hn_quant_act: leading dimension too small");
    REQUIRE(scale_strides_ok(M, per_row ? 1 : K / 128, s_rs, s_gs), HN_ERR_SHAPE,
            "hn_quant_act: scale strides (%lld, %lld) overlap", (long long)s_rs, (long long)s_gs);
    REQUIRE(M <= 0x7fffffffLL, HN_ERR_SHAPE, "hn_quant_act: M too large");
    REQUIRE(al16(x) && (ldx * dsize(x_dtype)) % 16 == 0 && al16(q) && ldq % 16 == 0, HN_ERR_ALIGN,
            "hn_quant_act: x/q must be 16-byte aligned with 16-byte row pitch");
    if (M == 0) return HN_OK;
    CHECK_DEVICE(x);
    return launched(launch_quant_act(x, ldx, x_dtype, M, K, kind, flags, q, ldq, s, s_rs, s_gs, (cudaStream_t)stream),
                    "hn_quant_act launch");
}

int hn_block_gemm(const void *qa, int64_t lda, const float *sa, int64_t sa_rs, int64_t sa_gs, int sa_mode,
                  const void *qw, int64_t ldw, const float *sw, int64_t sw_rs, int64_t sw_gs, int sw_mode,
                  const void *bias, int bias_dtype, void *out, int64_t ldo, int out_dtype, float *qs, int64_t qs_rs,
                  int64_t qs_gs, int64_t M, int64_t N, int64_t K, int kind, int epilogue, void *stream) {
    REQUIRE(qa && sa && qw && sw && out, HN_ERR_ARG, "hn_block_gemm: null pointer");
    REQUIRE(kind == HN_KIND_INT8 || kind == HN_KIND_FP8E4M3, HN_ERR_ARG, "hn_block_gemm: unknown kind %d", kind);
    REQUIRE(sa_mode == HN_SCALE_GROUP || sa_mode == HN_SCALE_ROW, HN_ERR_ARG, "hn_block_gemm: bad sa_mode %d", sa_mode);
    REQUIRE(sw_mode >= HN_SCALE_GROUP && sw_mode <= HN_SCALE_BLOCK, HN_ERR_ARG, "hn_block_gemm: bad sw_mode %d", sw_mode);
    REQUIRE(epilogue >= HN_EPI_NONE && epilogue <= HN_EPI_GELU_QUANT, HN_ERR_ARG, "hn_block_gemm: bad epilogue %d", epilogue);
    REQUIRE(M >= 0 && N > 0 && K > 0 && K % 128 == 0, HN_ERR_SHAPE,
            "hn_block_gemm: need K %% 128 == 0, N > 0 (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
    REQUIRE(M < (1LL << 31) && N < (1LL << 31) && K < (1LL << 31), HN_ERR_SHAPE, "hn_block_gemm: dimension too large");
    // both scales per row: the tensor core sums all of K in one int32 accumulator, |sum| <= K * 128 * 128
    REQUIRE(!(kind == HN_KIND_INT8 && sa_mode == HN_SCALE_ROW && sw_mode == HN_SCALE_ROW) || K <= HN_ROW_MODE_MAX_K,
            HN_ERR_SHAPE, "hn_block_gemm: int8 with per-row scales on both sides needs K <= %d (int32 accumulator; K=%lld)",
            HN_ROW_MODE_MAX_K, (long long)K);
    REQUIRE(lda >= K && ldw >= K && ldo >= N, HN_ERR_SHAPE, "hn_block_gemm: leading dimension too small");
    REQUIRE(sa_mode != HN_SCALE_GROUP || scale_strides_ok(M, K / 128, sa_rs, sa_gs), HN_ERR_SHAPE,
            "hn_block_gemm: activation scale strides overlap");
    REQUIRE(sw_mode != HN_SCALE_GROUP || scale_strides_ok(N, K / 128, sw_rs, sw_gs), HN_ERR_SHAPE,
            "hn_block_gemm: weight scale strides overlap");
    REQUIRE(sw_mode != HN_SCALE_BLOCK || scale_strides_ok(cdiv(N, 128), K / 128, sw_rs, sw_gs), HN_ERR_SHAPE,
            "hn_block_gemm: weight block scale strides overlap");
    REQUIRE(sa_mode != HN_SCALE_ROW || sa_rs >= 1, HN_ERR_SHAPE, "hn_block_gemm: sa_rs < 1");
    REQUIRE(sw_mode != HN_SCALE_ROW || sw_rs >= 1, HN_ERR_SHAPE, "hn_block_gemm: sw_rs < 1");
    REQUIRE(al16(qa) && al16(qw) && lda % 16 == 0 && ldw % 16 == 0, HN_ERR_ALIGN,
            "hn_block_gemm: qa/qw must be 16-byte aligned with row pitch a multiple of 16");
    if (epilogue == HN_EPI_GELU_QUANT) {
        REQUIRE(qs != nullptr, HN_ERR_ARG, "hn_block_gemm: gelu_quant needs qs");
        REQUIRE(N % 128 == 0, HN_ERR_SHAPE, "hn_block_gemm: gelu_quant needs N %% 128 == 0");
        REQUIRE(scale_strides_ok(M, N / 128, qs_rs, qs_gs), HN_ERR_SHAPE, "hn_block_gemm: qs strides overlap");
        REQUIRE(al16(out) && ldo % 16 == 0, HN_ERR_ALIGN, "hn_block_gemm: int8 output must be 16-byte aligned");
    } else if (epilogue == HN_EPI_GELU) {
        REQUIRE(out_dtype == HN_DTYPE_BF16, HN_ERR_UNSUPPORTED, "hn_block_gemm: gelu output is bf16");
    } else {
        REQUIRE(out_dtype >= HN_DTYPE_BF16 && out_dtype <= HN_DTYPE_INT32, HN_ERR_ARG, "hn_block_gemm: bad out_dtype %d", out_dtype);
    }
    if (out_dtype == HN_DTYPE_INT32)
        REQUIRE(kind == HN_KIND_INT8 && sa_mode == HN_SCALE_ROW && sw_mode == HN_SCALE_ROW && bias == nullptr &&
                    epilogue == HN_EPI_NONE,
                HN_ERR_UNSUPPORTED, "hn_block_gemm: int32 output is the raw int8 accumulator (row scales, no bias)");
    if (bias) REQUIRE(bias_dtype == HN_DTYPE_BF16 || bias_dtype == HN_DTYPE_FP16 || bias_dtype == HN_DTYPE_FP32,
                      HN_ERR_ARG, "hn_block_gemm: bad bias dtype %d", bias_dtype);
    // the epilogue reads the bias 8 columns at a time with 16-byte loads wherever 8 columns are in range
    if (bias) REQUIRE(al16(bias), HN_ERR_ALIGN, "hn_block_gemm: bias must be 16-byte aligned");
    if (M == 0) return HN_OK;
    CHECK_DEVICE(qa);
    GemmArgs a;
    a.qa = qa; a.lda = lda; a.sa = sa; a.sa_rs = sa_rs; a.sa_gs = sa_gs; a.sa_mode = sa_mode;
    a.qw = qw; a.ldw = ldw; a.sw = sw; a.sw_rs = sw_rs; a.sw_gs = sw_gs; a.sw_mode = sw_mode;
    a.bias = bias; a.bias_dtype = bias_dtype;
    a.out = out; a.ldo = ldo; a.out_dtype = out_dtype; a.qs = qs; a.qs_rs = qs_rs; a.qs_gs = qs_gs;
    a.M = M; a.N = N; a.K = K; a.kind = kind; a.epilogue = epilogue;
    a.sm_reserve = gemm_sm_reserve();
    const char *msg = nullptr;
    cudaError_t e = launch_block_gemm(a, (cudaStream_t)stream, &msg);
    if (e != cudaSuccess && msg) return fail(HN_ERR_ALIGN, "hn_block_gemm: %s", msg);
    return launched(e, "hn_block_gemm launch");
}

static int ln_common(const void *x, const void *shift, const void *scale, int64_t B, int64_t L, int64_t D, int quant,
                     const char *name) {
    REQUIRE(x && shift && scale, HN_ERR_ARG, "%s: null pointer", name);
    REQUIRE(B > 0 && L >= 0 && D > 0 && D <= 16384, HN_ERR_SHAPE, "%s: bad shape B=%lld L=%lld D=%lld", name,
            (long long)B, (long long)L, (long long)D);
    REQUIRE(quant ? D % 128 == 0 : D % 16 == 0, HN_ERR_SHAPE, "%s: D %% %d != 0", name, quant ? 128 : 16);
    REQUIRE(B * L < (1LL << 31), HN_ERR_SHAPE, "%s: too many rows", name);
    REQUIRE(al16(x) && al16(shift) && al16(scale), HN_ERR_ALIGN, "%s: inputs must be 16-byte aligned", name);
    return HN_OK;
}

int hn_adaln_quant(const void *x, const void *shift, const void *scale, int64_t B, int64_t L, int64_t D, float eps,
                   int8_t *q, float *s, int64_t s_rs, int64_t s_gs, void *stream) {
    int rc = ln_common(x, shift, scale, B, L, D, 1, "hn_adaln_quant");
    if (rc) return rc;
    REQUIRE(q && s && al16(q), HN_ERR_ARG, "hn_adaln_quant: null or misaligned output");
    REQUIRE(scale_strides_ok(B * L, D / 128, s_rs, s_gs), HN_ERR_SHAPE, "hn_adaln_quant: scale strides overlap");
    if (L == 0) return HN_OK;
    CHECK_DEVICE(x);
    return launched(launch_ln_row(1, x, nullptr, nullptr, shift, scale, B, L, D, eps, nullptr, q, s, s_rs, s_gs,
                                  (cudaStream_t)stream),
                    "hn_adaln_quant launch");
}

int hn_adaln(const void *x, const void *shift, const void *scale, int64_t B, int64_t L, int64_t D, float eps, void *y,
             void *stream) {
    int rc = ln_common(x, shift, scale, B, L, D, 0, "hn_adaln");
    if (rc) return rc;
    REQUIRE(y && al16(y), HN_ERR_ARG, "hn_adaln: null or misaligned output");
    if (L == 0) return HN_OK;
    CHECK_DEVICE(x);
    return launched(launch_ln_row(0, x, nullptr, nullptr, shift, scale, B, L, D, eps, y, nullptr, nullptr, 0, 0,
                                  (cudaStream_t)stream),
                    "hn_adaln launch");
}

int hn_gated_residual_adaln_quant(const void *x, const void *y, const void *gate, const void *shift, const void *scale,
                                  int64_t B, int64_t L, int64_t D, float eps, void *out, int8_t *q, float *s,
                                  int64_t s_rs, int64_t s_gs, void *stream) {
    int rc = ln_common(x, shift, scale, B, L, D, 1, "hn_gated_residual_adaln_quant");
    if (rc) return rc;
    REQUIRE(y && gate && out && q && s, HN_ERR_ARG, "hn_gated_residual_adaln_quant: null pointer");
    REQUIRE(al16(y) && al16(gate) && al16(out) && al16(q), HN_ERR_ALIGN,
            "hn_gated_residual_adaln_quant: buffers must be 16-byte aligned");
    REQUIRE(scale_strides_ok(B * L, D / 128, s_rs, s_gs), HN_ERR_SHAPE,
            "hn_gated_residual_adaln_quant: scale strides overlap");
    if (L == 0) return HN_OK;
    CHECK_DEVICE(x);
    return launched(launch_ln_row(2, x, y, gate, shift, scale, B, L, D, eps, out, q, s, s_rs, s_gs, (cudaStream_t)stream),
                    "hn_gated_residual_adaln_quant launch");
}

int hn_gated_residual(const void *x, const void *y, const void *gate, int64_t B, int64_t L, int64_t D, void *out,
                      void *stream) {
    REQUIRE(x && y && gate && out, HN_ERR_ARG, "hn_gated_residual: null pointer");
    REQUIRE(B > 0 && L >= 0 && D > 0 && D % 8 == 0, HN_ERR_SHAPE, "hn_gated_residual: need D %% 8 == 0");
    REQUIRE(al16(x) && al16(y) && al16(gate) && al16(out), HN_ERR_ALIGN, "hn_gated_residual: buffers must be 16-byte aligned");
    if (L == 0) return HN_OK;
    CHECK_DEVICE(x);
    return launched(launch_gated_residual(x, y, gate, B, L, D, out, (cudaStream_t)stream), "hn_gated_residual launch");
}

static int qk_common(const void *x, int64_t row_stride, const void *w, const float *cos, const float *sin, int64_t B,
                     int64_t L, int64_t H, int64_t D, const void *y) {
    REQUIRE(x && w && y, HN_ERR_ARG, "hn_qk_norm_rope: null pointer");
    REQUIRE((cos == nullptr) == (sin == nullptr), HN_ERR_ARG, "hn_qk_norm_rope: cos and sin must both be given or both NULL");
    REQUIRE(D == 128, HN_ERR_UNSUPPORTED, "hn_qk_norm_rope: head dim %lld (kernels are built for 128)", (long long)D);
    REQUIRE(B > 0 && L >= 0 && H > 0 && row_stride >= H * D, HN_ERR_SHAPE, "hn_qk_norm_rope: bad shape/stride");
    REQUIRE(al16(x) && row_stride % 8 == 0 && al16(w) && al16(y), HN_ERR_ALIGN,
            "hn_qk_norm_rope: x/w/y must be 16-byte aligned with a row stride that is a multiple of 8");
    REQUIRE(cos == nullptr || (al16(cos) && al16(sin)), HN_ERR_ALIGN, "hn_qk_norm_rope: cos/sin must be 16-byte aligned");
    return HN_OK;
}

int hn_qk_norm_rope(const void *x, int64_t row_stride, const void *weight, const float *cos, const float *sin,
                    int64_t B, int64_t L, int64_t H, int64_t D, float eps, void *y, void *stream) {
    int rc = qk_common(x, row_stride, weight, cos, sin, B, L, H, D, y);
    if (rc) return rc;
    if (L == 0) return HN_OK;
    CHECK_DEVICE(x);
    return launched(launch_qk_norm_rope(1, x, nullptr, row_stride, weight, nullptr, cos, sin, B, L, H, eps, y, nullptr,
                                        nullptr, nullptr, (cudaStream_t)stream),
                    "hn_qk_norm_rope launch");
}

int hn_qk_norm_rope_kv(const void *x, int64_t row_stride, const void *weight, const float *cos, const float *sin,
                       int64_t B, int64_t L, int64_t H, int64_t D, float eps, void *y, int8_t *q, float *s,
                       void *stream) {
    int rc = qk_common(x, row_stride, weight, cos, sin, B, L, H, D, y);
    if (rc) return rc;
    REQUIRE(q && s, HN_ERR_ARG, "hn_qk_norm_rope_kv: null pointer");
    REQUIRE(al16(q) && (reinterpret_cast<uintptr_t>(s) & 3) == 0, HN_ERR_ALIGN, "hn_qk_norm_rope_kv: misaligned buffer");
    if (L == 0) return HN_OK;
    CHECK_DEVICE(x);
    return launched(launch_qk_norm_rope(1, x, nullptr, row_stride, weight, nullptr, cos, sin, B, L, H, eps, y, nullptr,
                                        q, s, (cudaStream_t)stream),
                    "hn_qk_norm_rope_kv launch");
}

int hn_qk_norm_rope2(const void *xq, const void *xk, int64_t row_stride, const void *wq, const void *wk,
                     const float *cos, const float *sin, int64_t B, int64_t L, int64_t H, int64_t D, float eps,
                     void *yq, void *yk, void *stream) {
    int rc = qk_common(xq, row_stride, wq, cos, sin, B, L, H, D, yq);
    if (rc) return rc;
    rc = qk_common(xk, row_stride, wk, cos, sin, B, L, H, D, yk);
    if (rc) return rc;
    if (L == 0) return HN_OK;
    CHECK_DEVICE(xq);
    return launched(launch_qk_norm_rope(2, xq, xk, row_stride, wq, wk, cos, sin, B, L, H, eps, yq, yk, nullptr, nullptr,
                                        (cudaStream_t)stream),
                    "hn_qk_norm_rope2 launch");
}

int hn_pixelumm_qk(const void *x, int64_t row_stride, const void *weight_t, const void *weight_hw, const float *cos,
                   const float *sin, int64_t N, int64_t H, int64_t D, float eps, void *y, void *stream) {
    REQUIRE(x && weight_t && weight_hw && cos && sin && y, HN_ERR_ARG, "hn_pixelumm_qk: null pointer");
    REQUIRE(D == 128, HN_ERR_UNSUPPORTED, "hn_pixelumm_qk: head dim %lld (kernels are built for 128)", (long long)D);
    REQUIRE(N >= 0 && H > 0 && row_stride >= H * D, HN_ERR_SHAPE, "hn_pixelumm_qk: bad shape/stride");
    REQUIRE(al8(x) && row_stride % 4 == 0 && al8(weight_t) && al8(weight_hw) && al16(cos) && al16(sin) && al8(y),
            HN_ERR_ALIGN, "hn_pixelumm_qk: misaligned buffer");
    if (N == 0) return HN_OK;
    CHECK_DEVICE(x);
    return launched(launch_pixelumm_qk(x, row_stride, weight_t, weight_hw, cos, sin, N, H, eps, y, (cudaStream_t)stream),
                    "hn_pixelumm_qk launch");
}

int hn_quantize_kv(const void *x, int64_t rows, int64_t D, int8_t *q, float *s, void *stream) {
    REQUIRE(D > 0 && D % 128 == 0, HN_ERR_SHAPE, "hn_quantize_kv: need D %% 128 == 0");
    return hn_quant_act(x, D, HN_DTYPE_BF16, rows, D, HN_KIND_INT8, D == 128 ? 0 : 1, q, D, s, 1, 1, stream);
}

int hn_dequantize_kv(const int8_t *q, const float *s, int64_t rows, int64_t D, void *y, void *stream) {
    REQUIRE(q && s && y, HN_ERR_ARG, "hn_dequantize_kv: null pointer");
    REQUIRE(rows >= 0 && D > 0 && D % 16 == 0, HN_ERR_SHAPE, "hn_dequantize_kv: need D %% 16 == 0 (D=%lld)", (long long)D);
    REQUIRE(al16(q) && al16(y) && (reinterpret_cast<uintptr_t>(s) & 3) == 0, HN_ERR_ALIGN,
            "hn_dequantize_kv: misaligned buffer");
    if (rows == 0) return HN_OK;
    CHECK_DEVICE(q);
    return launched(launch_dequant_kv(q, s, rows, D, y, (cudaStream_t)stream), "hn_dequantize_kv launch");
}

int hn_rmsnorm_quant(const void *x, int64_t ldx, const void *weight, int64_t rows, int64_t D, float eps, int kind,
                     void *q, int64_t ldq, float *s, int64_t s_rs, int64_t s_gs, void *stream) {
    REQUIRE(x && weight && q && s, HN_ERR_ARG, "hn_rmsnorm_quant: null pointer");
    REQUIRE(kind == HN_KIND_INT8 || kind == HN_KIND_FP8E4M3, HN_ERR_ARG, "hn_rmsnorm_quant: unknown kind %d", kind);
    REQUIRE(rows >= 0 && D > 0 && D % 128 == 0 && D <= 16384, HN_ERR_SHAPE,
            "hn_rmsnorm_quant: need D %% 128 == 0 and D <= 16384 (D=%lld)", (long long)D);
    REQUIRE(rows < (1LL << 31) && ldx >= D && ldq >= D, HN_ERR_SHAPE, "hn_rmsnorm_quant: bad rows or leading dimension");
    REQUIRE(scale_strides_ok(rows, D / 128, s_rs, s_gs), HN_ERR_SHAPE, "hn_rmsnorm_quant: scale strides overlap");
    REQUIRE(al16(x) && ldx % 8 == 0 && al16(weight) && al16(q) && ldq % 16 == 0, HN_ERR_ALIGN,
            "hn_rmsnorm_quant: x/weight/q must be 16-byte aligned with 16-byte row pitches");
    if (rows == 0) return HN_OK;
    CHECK_DEVICE(x);
    return launched(launch_rmsnorm_quant(x, ldx, weight, rows, D, eps, kind, q, ldq, s, s_rs, s_gs, (cudaStream_t)stream),
                    "hn_rmsnorm_quant launch");
}

int hn_silu_mul_quant(const void *g, int64_t ldg, const void *u, int64_t ldu, int64_t rows, int64_t I, int kind,
                      void *q, int64_t ldq, float *s, int64_t s_rs, int64_t s_gs, void *stream) {
    REQUIRE(g && u && q && s, HN_ERR_ARG, "hn_silu_mul_quant: null pointer");
    REQUIRE(kind == HN_KIND_INT8 || kind == HN_KIND_FP8E4M3, HN_ERR_ARG, "hn_silu_mul_quant: unknown kind %d", kind);
    REQUIRE(rows >= 0 && I > 0 && I % 128 == 0, HN_ERR_SHAPE, "hn_silu_mul_quant: need I %% 128 == 0 (I=%lld)", (long long)I);
    REQUIRE(ldg >= I && ldu >= I && ldq >= I, HN_ERR_SHAPE, "hn_silu_mul_quant: leading dimension too small");
    REQUIRE(scale_strides_ok(rows, I / 128, s_rs, s_gs), HN_ERR_SHAPE, "hn_silu_mul_quant: scale strides overlap");
    REQUIRE(al16(g) && al16(u) && ldg % 8 == 0 && ldu % 8 == 0 && al16(q) && ldq % 16 == 0, HN_ERR_ALIGN,
            "hn_silu_mul_quant: g/u/q must be 16-byte aligned with 16-byte row pitches");
    if (rows == 0) return HN_OK;
    CHECK_DEVICE(g);
    return launched(launch_silu_mul_quant(g, ldg, u, ldu, rows, I, kind, q, ldq, s, s_rs, s_gs, (cudaStream_t)stream),
                    "hn_silu_mul_quant launch");
}

int hn_add_rmsnorm_quant(const void *x, int64_t ldx, const void *r, int64_t ldr, const void *weight, int64_t rows,
                         int64_t D, float eps, int kind, int flags, void *out, int64_t ldo, void *q, int64_t ldq,
                         float *s, int64_t s_rs, int64_t s_gs, void *stream) {
    REQUIRE(rows == 0 || (x && r && weight && out && q && s), HN_ERR_ARG, "hn_add_rmsnorm_quant: null pointer");
    REQUIRE(kind == HN_KIND_INT8 || kind == HN_KIND_FP8E4M3, HN_ERR_ARG, "hn_add_rmsnorm_quant: unknown kind %d", kind);
    REQUIRE((flags & ~HN_QUANT_PER_ROW) == 0, HN_ERR_ARG, "hn_add_rmsnorm_quant: unknown flags %d", flags);
    const bool per_row = (flags & HN_QUANT_PER_ROW) != 0;
    REQUIRE(rows >= 0 && rows < (1LL << 31) && D > 0 && D % 128 == 0 && D <= 16384, HN_ERR_SHAPE,
            "hn_add_rmsnorm_quant: need D %% 128 == 0 and D <= 16384 (rows=%lld D=%lld)", (long long)rows, (long long)D);
    if (rows == 0) return HN_OK;
    REQUIRE(ldx >= D && ldr >= D && ldo >= D && ldq >= D, HN_ERR_SHAPE, "hn_add_rmsnorm_quant: leading dimension too small");
    REQUIRE(scale_strides_ok(rows, per_row ? 1 : D / 128, s_rs, s_gs), HN_ERR_SHAPE,
            "hn_add_rmsnorm_quant: scale strides overlap");
    REQUIRE(al16(x) && al16(r) && al16(weight) && al16(out) && al16(q) && ldx % 8 == 0 && ldr % 8 == 0 && ldo % 8 == 0 &&
                ldq % 16 == 0, HN_ERR_ALIGN, "hn_add_rmsnorm_quant: 16-byte aligned pointers and row pitches needed");
    CHECK_DEVICE(x);
    return launched(launch_add_rmsnorm_quant(x, ldx, r, ldr, weight, rows, D, eps, kind, per_row, out, ldo, q, ldq, s, s_rs,
                                             s_gs, (cudaStream_t)stream), "hn_add_rmsnorm_quant launch");
}

// the cache's own checks, then `a` filled in
static int cache_args(const hn_kv_cache *c, const char *what, CacheArgs &a) {
    REQUIRE(c && c->k && c->v && c->table && c->lengths && c->refs && c->failed, HN_ERR_ARG, "%s: null pointer in the cache", what);
    REQUIRE((c->k_scale == nullptr) == (c->v_scale == nullptr), HN_ERR_ARG, "%s: one of the two scale pools is missing", what);
    REQUIRE(c->layers > 0 && c->pages > 0 && c->heads > 0 && c->slots > 0 && c->width > 0, HN_ERR_SHAPE,
            "%s: layers, pages, heads, slots and width must be positive", what);
    REQUIRE(c->page >= 16 && c->page % 16 == 0, HN_ERR_SHAPE, "%s: the page must be a multiple of 16 tokens (%lld)", what,
            (long long)c->page);
    const int64_t most = 0x7fffffff;
    REQUIRE(c->layers <= most && c->pages <= most / 4 && c->heads <= 65536 && c->slots <= most / 4 && c->page <= most &&
                c->width <= most / c->page && c->heads * c->page <= most / 256 && c->pages <= most / c->heads / (c->page / 16), HN_ERR_SHAPE, "%s: the cache is too large", what);
    REQUIRE(al16(c->k) && al16(c->v) && al16(c->k_scale) && al16(c->v_scale), HN_ERR_ALIGN,
            "%s: the pools must be 16-byte aligned", what);
    a.k = c->k; a.v = c->v; a.ks = c->k_scale; a.vs = c->v_scale;
    a.layers = (int)c->layers; a.heads = (int)c->heads;
    a.meta.table = c->table; a.meta.lengths = c->lengths; a.meta.refs = c->refs; a.meta.failed = c->failed;
    a.meta.refused = c->refused; a.meta.epoch = c->epoch;
    a.meta.slots = (int)c->slots; a.meta.width = (int)c->width; a.meta.pages = (int)c->pages; a.meta.page = (int)c->page;
    return HN_OK;
}
// at most so many requests a call (their number is a grid or a loop count of int)
constexpr int64_t MAX_REQUESTS = 1 << 24;

int hn_cache_workspace(const hn_kv_cache *cache, int64_t n, int64_t *words_host) {
    CacheArgs a;
    if (int rc = cache_args(cache, "hn_cache_workspace", a)) return rc;
    REQUIRE(words_host && n >= 0 && n <= MAX_REQUESTS, HN_ERR_ARG, "hn_cache_workspace: bad arguments");
    const int64_t requests = cache->slots + cache->pages + 4 * n, moves = 4 + 3 * cache->pages;
    *words_host = requests > moves ? requests : moves;
    t_last_error.clear();
    return HN_OK;
}

int hn_cache_extend(const hn_kv_cache *cache, const int32_t *rows, int64_t n, int64_t tokens, int32_t *ws, void *stream) {
    CacheArgs a;
    if (int rc = cache_args(cache, "hn_cache_extend", a)) return rc;
    REQUIRE(n >= 0 && n <= MAX_REQUESTS && tokens >= 0 && tokens <= 0x3fffffff, HN_ERR_SHAPE,
            "hn_cache_extend: bad count (n=%lld tokens=%lld)", (long long)n, (long long)tokens);
    if (n == 0) return HN_OK;
    REQUIRE(rows && ws && cache->refused, HN_ERR_ARG, "hn_cache_extend: null pointer");
    REQUIRE(cache->epoch != 0, HN_ERR_ARG, "hn_cache_extend: the cache's epoch is 0");
    CHECK_DEVICE(cache->k);
    return launched(launch_cache_extend(a.meta, rows, (int)n, (int)tokens, ws, (cudaStream_t)stream), "hn_cache_extend launch");
}

int hn_cache_append(const hn_kv_cache *cache, int64_t layer, const void *k, int64_t k_bs, int64_t k_ts, int64_t k_hs,
                    const void *v, int64_t v_bs, int64_t v_ts, int64_t v_hs, const int32_t *rows, int64_t B, int64_t n,
                    void *stream) {
    CacheArgs a;
    if (int rc = cache_args(cache, "hn_cache_append", a)) return rc;
    REQUIRE(layer >= 0 && layer < cache->layers, HN_ERR_SHAPE, "hn_cache_append: layer %lld of %lld", (long long)layer,
            (long long)cache->layers);
    REQUIRE(B >= 0 && n >= 0 && B <= MAX_REQUESTS && n <= 0x3fffffff, HN_ERR_SHAPE, "hn_cache_append: bad count");
    if (B == 0 || n == 0) return HN_OK;
    REQUIRE(k && v && rows, HN_ERR_ARG, "hn_cache_append: null pointer");
    REQUIRE(al16(k) && al16(v) && (k_bs | k_ts | k_hs | v_bs | v_ts | v_hs) % 8 == 0, HN_ERR_ALIGN,
            "hn_cache_append: k and v need 16-byte aligned rows of 128");
    REQUIRE(cache->refused, HN_ERR_ARG, "hn_cache_append: null pointer in the cache");
    REQUIRE(cache->epoch != 0, HN_ERR_ARG, "hn_cache_append: the cache's epoch is 0");
    CHECK_DEVICE(k);
    return launched(launch_cache_append(a, (int)layer, k, k_bs, k_ts, k_hs, v, v_bs, v_ts, v_hs, rows, (int)B, (int)n,
                                        (cudaStream_t)stream), "hn_cache_append launch");
}

int hn_cache_free(const hn_kv_cache *cache, const int32_t *rows, int64_t n, void *stream) {
    CacheArgs a;
    if (int rc = cache_args(cache, "hn_cache_free", a)) return rc;
    REQUIRE(n >= 0 && n <= MAX_REQUESTS, HN_ERR_SHAPE, "hn_cache_free: bad count %lld", (long long)n);
    if (n == 0) return HN_OK;
    REQUIRE(rows && cache->refused, HN_ERR_ARG, "hn_cache_free: null pointer");
    CHECK_DEVICE(cache->k);
    return launched(launch_cache_free(a.meta, rows, (int)n, (cudaStream_t)stream), "hn_cache_free launch");
}

int hn_cache_fork(const hn_kv_cache *cache, const int32_t *parents, const int32_t *children, int64_t n, int32_t *ws,
                  void *stream) {
    CacheArgs a;
    if (int rc = cache_args(cache, "hn_cache_fork", a)) return rc;
    REQUIRE(n >= 0 && n <= MAX_REQUESTS, HN_ERR_SHAPE, "hn_cache_fork: bad count %lld", (long long)n);
    if (n == 0) return HN_OK;
    REQUIRE(parents && children && ws && cache->refused, HN_ERR_ARG, "hn_cache_fork: null pointer");
    CHECK_DEVICE(cache->k);
    return launched(launch_cache_fork(a, parents, children, (int)n, ws, (cudaStream_t)stream), "hn_cache_fork launch");
}

int hn_cache_compact(const hn_kv_cache *cache, int32_t *ws, void *stream) {
    CacheArgs a;
    if (int rc = cache_args(cache, "hn_cache_compact", a)) return rc;
    REQUIRE(ws, HN_ERR_ARG, "hn_cache_compact: null pointer");
    CHECK_DEVICE(cache->k);
    return launched(launch_cache_compact(a, ws, (cudaStream_t)stream), "hn_cache_compact launch");
}

int hn_cache_copy(const hn_kv_cache *cache, const int32_t *src, const int32_t *dst, int64_t n, void *stream) {
    CacheArgs a;
    if (int rc = cache_args(cache, "hn_cache_copy", a)) return rc;
    REQUIRE(n >= 0 && n <= MAX_REQUESTS, HN_ERR_SHAPE, "hn_cache_copy: bad count %lld", (long long)n);
    if (n == 0) return HN_OK;
    REQUIRE(src && dst, HN_ERR_ARG, "hn_cache_copy: null pointer");
    CHECK_DEVICE(cache->k);
    return launched(launch_cache_copy(a, src, dst, (int)n, (cudaStream_t)stream), "hn_cache_copy launch");
}

// rows of `width` elements at b * bs + l * ls + h * hs that do not overlap: each stride is past what the smaller ones reach (a
// dimension of one has none)
static bool rows_apart(int64_t B, int64_t bs, int64_t Lq, int64_t ls, int64_t H, int64_t hs, int64_t width = 128) {
    int64_t n[3] = {B, Lq, H}, s[3] = {bs < 0 ? -bs : bs, ls < 0 ? -ls : ls, hs < 0 ? -hs : hs};
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2 - i; ++j)
            if (s[j] > s[j + 1]) { std::swap(s[j], s[j + 1]); std::swap(n[j], n[j + 1]); }
    int64_t reach = width;
    for (int i = 0; i < 3; ++i) {
        if (n[i] == 1) continue;
        if (s[i] < reach) return false;
        reach += s[i] * (n[i] - 1);
    }
    return true;
}

// the shape checks of hn_paged_attention and of its workspace
static int paged_args(const hn_kv_cache *cache, const char *what, int64_t B, int64_t Lq, int64_t H, int64_t shared, int causal,
                      PagedAttnArgs &a) {
    if (int rc = cache_args(cache, what, a.cache)) return rc;
    REQUIRE(B >= 0 && B <= 4096 && Lq >= 0 && H > 0 && H % cache->heads == 0, HN_ERR_SHAPE,
            "%s: need 0 <= B <= 4096 and H a multiple of the cache's %lld heads (B=%lld Lq=%lld H=%lld)", what,
            (long long)cache->heads, (long long)B, (long long)Lq, (long long)H);
    REQUIRE(H <= 65536 && Lq <= (1LL << 24) && B * Lq * H <= (1LL << 29), HN_ERR_SHAPE, "%s: too many queries", what);
    REQUIRE(shared >= 0 && shared % cache->page == 0 && shared <= cache->width * cache->page, HN_ERR_SHAPE,
            "%s: shared must be whole pages within the table (%lld, page %lld)", what, (long long)shared, (long long)cache->page);
    REQUIRE(causal == 0 || causal == 1, HN_ERR_ARG, "%s: causal is 0 or 1", what);
    a.B = (int)B; a.Lq = (int)Lq; a.H = (int)H; a.shared = (int)shared; a.causal = causal;
    return HN_OK;
}

int hn_paged_attention_workspace(const hn_kv_cache *cache, int64_t B, int64_t Lq, int64_t H, int64_t shared, int causal,
                                 int64_t *bytes_host) {
    PagedAttnArgs a;
    if (int rc = paged_args(cache, "hn_paged_attention_workspace", B, Lq, H, shared, causal, a)) return rc;
    REQUIRE(bytes_host, HN_ERR_ARG, "hn_paged_attention_workspace: null pointer");
    *bytes_host = B == 0 || Lq == 0 ? 0 : paged_attention_ws(a);
    t_last_error.clear();
    return HN_OK;
}

int hn_paged_attention(const hn_kv_cache *cache, int64_t layer, const void *q, int64_t q_bs, int64_t q_ls, int64_t q_hs,
                       const int32_t *rows, int64_t B, int64_t Lq, int64_t H, int64_t D, int64_t shared, int causal,
                       float scale, void *out, int64_t o_bs, int64_t o_ls, int64_t o_hs, float *lse, void *ws,
                       int64_t ws_bytes, void *stream) {
    PagedAttnArgs a;
    if (int rc = paged_args(cache, "hn_paged_attention", B, Lq, H, shared, causal, a)) return rc;
    REQUIRE(D == 128, HN_ERR_UNSUPPORTED, "hn_paged_attention: head dim %lld (128 is supported)", (long long)D);
    REQUIRE(layer >= 0 && layer < cache->layers, HN_ERR_SHAPE, "hn_paged_attention: layer %lld of %lld", (long long)layer,
            (long long)cache->layers);
    if (B == 0 || Lq == 0) return HN_OK;
    REQUIRE(std::isfinite(scale), HN_ERR_ARG, "hn_paged_attention: the scale is not a finite number");
    REQUIRE(q && rows && out && ws, HN_ERR_ARG, "hn_paged_attention: null pointer");
    REQUIRE(al16(q) && al16(out) && al16(ws) && (q_bs | q_ls | q_hs | o_bs | o_ls | o_hs) % 8 == 0, HN_ERR_ALIGN,
            "hn_paged_attention: q, out and ws must be 16-byte aligned, strides multiples of 8 elements");
    REQUIRE(rows_apart(B, o_bs, Lq, o_ls, H, o_hs), HN_ERR_SHAPE, "hn_paged_attention: the rows of out overlap");
    CHECK_DEVICE(q);
    const int64_t tokens = layer * cache->pages * cache->heads * cache->page;
    const int64_t row_bytes = cache->k_scale ? 128 : 256;
    a.cache.k = static_cast<uint8_t *>(cache->k) + tokens * row_bytes;
    a.cache.v = static_cast<uint8_t *>(cache->v) + tokens * row_bytes;
    if (cache->k_scale) { a.cache.ks += tokens; a.cache.vs += tokens; }
    a.q = q; a.q_bs = q_bs; a.q_ls = q_ls; a.q_hs = q_hs;
    a.out = out; a.o_bs = o_bs; a.o_ls = o_ls; a.o_hs = o_hs;
    a.lse = lse; a.rows = rows; a.scale = scale; a.ws = ws; a.ws_bytes = ws_bytes;
    const int64_t need = paged_attention_ws(a);
    REQUIRE(ws_bytes >= need, HN_ERR_ARG, "hn_paged_attention: the workspace has %lld bytes, %lld are needed",
            (long long)ws_bytes, (long long)need);
    return launched(launch_paged_attention(a, (cudaStream_t)stream), "hn_paged_attention launch");
}

int hn_quantize_fp8_block(const void *w, int w_dtype, int64_t N, int64_t K, void *q, float *s, void *stream) {
    REQUIRE(w && q && s, HN_ERR_ARG, "hn_quantize_fp8_block: null pointer");
    REQUIRE(w_dtype == HN_DTYPE_FP32 || w_dtype == HN_DTYPE_BF16, HN_ERR_ARG,
            "hn_quantize_fp8_block: w_dtype %d not fp32/bf16", w_dtype);
    REQUIRE(N >= 0 && K >= 0 && N % 128 == 0 && K % 128 == 0, HN_ERR_SHAPE,
            "hn_quantize_fp8_block: need N %% 128 == 0 and K %% 128 == 0 (N=%lld K=%lld)", (long long)N, (long long)K);
    REQUIRE(N / 128 <= 65535 && K / 128 <= 0x7fffffffLL, HN_ERR_SHAPE, "hn_quantize_fp8_block: too large");
    REQUIRE(al16(w) && al16(q) && (reinterpret_cast<uintptr_t>(s) & 3) == 0, HN_ERR_ALIGN, "hn_quantize_fp8_block: misaligned buffer");
    if (N == 0 || K == 0) return HN_OK;
    CHECK_DEVICE(w);
    return launched(launch_quant_fp8_block(w, w_dtype, N, K, q, s, (cudaStream_t)stream), "hn_quantize_fp8_block launch");
}

int hn_attention(const void *q, int64_t q_rs, int64_t q_hs, int64_t q_bs, const void *k, int64_t k_rs, int64_t k_hs,
                 int64_t k_bs, const void *v, int64_t v_rs, int64_t v_hs, int64_t v_bs, int64_t B, int64_t Lq,
                 int64_t Lk, int64_t H, int64_t D, float scale, void *out, int64_t o_rs, int64_t o_hs, int64_t o_bs,
                 int8_t *q8, float *s8, void *stream) {
    REQUIRE(q && k && v, HN_ERR_ARG, "hn_attention: null q/k/v");
    REQUIRE(out != nullptr || q8 != nullptr, HN_ERR_ARG, "hn_attention: no output (out and q8 both null)");
    REQUIRE((q8 == nullptr) == (s8 == nullptr), HN_ERR_ARG, "hn_attention: q8 and s8 go together");
    REQUIRE(D == 128, HN_ERR_UNSUPPORTED, "hn_attention: head dim %lld (128 supported)", (long long)D);
    REQUIRE(B >= 1 && H >= 1 && Lq >= 1 && Lk >= 1, HN_ERR_SHAPE, "hn_attention: empty shape B=%lld H=%lld Lq=%lld Lk=%lld",
            (long long)B, (long long)H, (long long)Lq, (long long)Lk);
    REQUIRE(B <= 65535 && H <= 65535 && Lq < (1LL << 31) && Lk < (1LL << 31) && B * Lq < (1LL << 31), HN_ERR_SHAPE,
            "hn_attention: too large");
    REQUIRE(std::isfinite(scale) && scale > 0.0f, HN_ERR_ARG, "hn_attention: scale must be positive and finite");
    const int64_t st_in[9] = {q_rs, q_hs, q_bs, k_rs, k_hs, k_bs, v_rs, v_hs, v_bs};
    for (int i = 0; i < 9; ++i)
        REQUIRE(st_in[i] >= 0 && st_in[i] % 8 == 0 && st_in[i] < (1LL << 38), HN_ERR_ALIGN,
                "hn_attention: input strides must be non-negative multiples of 8 elements");
    REQUIRE(al16(q) && al16(k) && al16(v), HN_ERR_ALIGN, "hn_attention: q/k/v must be 16-byte aligned");
    if (out != nullptr)
        REQUIRE(al16(out) && o_rs >= 0 && o_hs >= 0 && o_bs >= 0 && o_rs % 8 == 0 && o_hs % 8 == 0 && o_bs % 8 == 0,
                HN_ERR_ALIGN, "hn_attention: out must be 16-byte aligned with strides multiples of 8 elements");
    if (q8 != nullptr)
        REQUIRE(reinterpret_cast<uintptr_t>(q8) % 8 == 0 && reinterpret_cast<uintptr_t>(s8) % 4 == 0, HN_ERR_ALIGN,
                "hn_attention: q8 must be 8-byte and s8 4-byte aligned");
    CHECK_DEVICE(q);
    AttnArgs a;
    a.q = q; a.k = k; a.v = v;
    a.q_rs = q_rs; a.q_hs = q_hs; a.q_bs = q_bs; a.k_rs = k_rs; a.k_hs = k_hs; a.k_bs = k_bs;
    a.v_rs = v_rs; a.v_hs = v_hs; a.v_bs = v_bs;
    a.B = B; a.Lq = Lq; a.Lk = Lk; a.H = H; a.scale = scale;
    a.out = out; a.o_rs = o_rs; a.o_hs = o_hs; a.o_bs = o_bs; a.q8 = q8; a.s8 = s8;
    const char *msg = nullptr;
    cudaError_t e = launch_attention(a, (cudaStream_t)stream, &msg);
    if (e != cudaSuccess && msg) return fail(HN_ERR_ALIGN, "hn_attention: %s", msg);
    return launched(e, "hn_attention launch");
}

int hn_attn_merge(const void *const *parts, const float *const *lses, int64_t n, int64_t o_bs, int64_t o_qs,
                  int64_t o_hs, int64_t l_bs, int64_t l_hs, int64_t l_qs, int64_t B, int64_t Lq, int64_t H, int64_t D,
                  void *out, int64_t out_bs, int64_t out_qs, int64_t out_hs, int8_t *q8, float *s8, void *stream) {
    REQUIRE(parts && lses, HN_ERR_ARG, "hn_attn_merge: null piece arrays");
    REQUIRE(n >= 1 && n <= 16, HN_ERR_SHAPE, "hn_attn_merge: %lld pieces (1 to 16)", (long long)n);
    REQUIRE(out != nullptr || q8 != nullptr, HN_ERR_ARG, "hn_attn_merge: no output");
    REQUIRE((q8 == nullptr) == (s8 == nullptr), HN_ERR_ARG, "hn_attn_merge: q8 and s8 go together");
    REQUIRE(D == 128, HN_ERR_UNSUPPORTED, "hn_attn_merge: head dim %lld (128 supported)", (long long)D);
    REQUIRE(B >= 1 && Lq >= 0 && H >= 1 && B * Lq * H < (1LL << 40) && B * Lq < (1LL << 31), HN_ERR_SHAPE,
            "hn_attn_merge: bad shape");
    for (int64_t i = 0; i < n; ++i) {
        REQUIRE(parts[i] && lses[i], HN_ERR_ARG, "hn_attn_merge: null piece %lld", (long long)i);
        REQUIRE(reinterpret_cast<uintptr_t>(parts[i]) % 8 == 0 && reinterpret_cast<uintptr_t>(lses[i]) % 4 == 0,
                HN_ERR_ALIGN, "hn_attn_merge: piece %lld misaligned", (long long)i);
    }
    REQUIRE(o_bs % 4 == 0 && o_qs % 4 == 0 && o_hs % 4 == 0 && o_bs >= 0 && o_qs >= 0 && o_hs >= 0, HN_ERR_ALIGN,
            "hn_attn_merge: piece strides must be non-negative multiples of 4 elements");
    REQUIRE(l_bs >= 0 && l_hs >= 0 && l_qs >= 0, HN_ERR_ARG, "hn_attn_merge: negative log-sum-exp stride");
    if (out != nullptr)
        REQUIRE(reinterpret_cast<uintptr_t>(out) % 8 == 0 && out_bs % 4 == 0 && out_qs % 4 == 0 && out_hs % 4 == 0 &&
                    out_bs >= 0 && out_qs >= 0 && out_hs >= 0,
                HN_ERR_ALIGN, "hn_attn_merge: out must be 8-byte aligned with strides multiples of 4 elements");
    if (q8 != nullptr)
        REQUIRE(reinterpret_cast<uintptr_t>(q8) % 4 == 0 && reinterpret_cast<uintptr_t>(s8) % 4 == 0, HN_ERR_ALIGN,
                "hn_attn_merge: q8 / s8 must be 4-byte aligned");
    if (Lq == 0) return HN_OK;
    CHECK_DEVICE(parts[0]);
    MergeArgs a;
    a.parts = parts; a.lses = lses; a.n = n;
    a.o_bs = o_bs; a.o_qs = o_qs; a.o_hs = o_hs; a.l_bs = l_bs; a.l_hs = l_hs; a.l_qs = l_qs;
    a.B = B; a.Lq = Lq; a.H = H;
    a.out = out; a.out_bs = out_bs; a.out_qs = out_qs; a.out_hs = out_hs; a.q8 = q8; a.s8 = s8;
    return launched(launch_attn_merge(a, (cudaStream_t)stream), "hn_attn_merge launch");
}

} // extern "C"

// ---------------------------------------------------------------------------------------------------
// 4-bit linears, rotations

extern "C" {

static bool fp4_kind(int kind) { return kind == HN_KIND_MXFP4 || kind == HN_KIND_NVFP4; }
static bool float_dtype(int dt) { return dt == HN_DTYPE_BF16 || dt == HN_DTYPE_FP16 || dt == HN_DTYPE_FP32; }
static bool al4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

int hn_quantize_fp4(const void *x, int64_t ldx, int x_dtype, int64_t M, int64_t K, int kind, void *q, int64_t ldq, void *s,
                    float *r, void *stream) {
    REQUIRE(fp4_kind(kind), HN_ERR_ARG, "hn_quantize_fp4: unknown kind %d", kind);
    REQUIRE(float_dtype(x_dtype), HN_ERR_ARG, "hn_quantize_fp4: bad x_dtype %d", x_dtype);
    REQUIRE(M >= 0 && M <= 0x7fffff00LL && K > 0 && K <= (1LL << 30), HN_ERR_SHAPE,
            "hn_quantize_fp4: bad shape (M=%lld K=%lld)", (long long)M, (long long)K);
    if (M == 0) return HN_OK;
    REQUIRE(x && q && s && (kind == HN_KIND_MXFP4 || r), HN_ERR_ARG, "hn_quantize_fp4: null pointer");
    REQUIRE(ldx >= K && ldq >= cdiv(K, 32) * 16, HN_ERR_SHAPE, "hn_quantize_fp4: leading dimension too small");
    REQUIRE(reinterpret_cast<uintptr_t>(x) % dsize(x_dtype) == 0 && al16(q) && ldq % 16 == 0 && al16(s) && al4(r), HN_ERR_ALIGN,
            "hn_quantize_fp4: q and s need 16-byte aligned rows, x its type's alignment");
    CHECK_DEVICE(x);
    return launched(launch_quant_fp4(x, ldx, x_dtype, M, K, kind - HN_KIND_MXFP4, q, ldq, s, r, (cudaStream_t)stream),
                    "hn_quantize_fp4 launch");
}

int hn_dequantize_fp4(const void *q, int64_t ldq, const void *s, const float *r, int64_t M, int64_t K, int64_t Kp, int kind,
                      void *out, int64_t ldo, int out_dtype, void *stream) {
    REQUIRE(fp4_kind(kind), HN_ERR_ARG, "hn_dequantize_fp4: unknown kind %d", kind);
    REQUIRE(float_dtype(out_dtype), HN_ERR_ARG, "hn_dequantize_fp4: bad out_dtype %d", out_dtype);
    REQUIRE(M >= 0 && M <= 0x7fffff00LL && K > 0 && K <= Kp && Kp <= (1LL << 30) && Kp % 32 == 0, HN_ERR_SHAPE,
            "hn_dequantize_fp4: bad shape (M=%lld K=%lld of %lld)", (long long)M, (long long)K, (long long)Kp);
    if (M == 0) return HN_OK;
    REQUIRE(q && s && out && (kind == HN_KIND_MXFP4 || r), HN_ERR_ARG, "hn_dequantize_fp4: null pointer");
    REQUIRE(ldo >= K && ldq >= Kp / 2, HN_ERR_SHAPE, "hn_dequantize_fp4: leading dimension too small");
    REQUIRE(al16(q) && ldq % 16 == 0 && al16(s) && al4(r) && reinterpret_cast<uintptr_t>(out) % dsize(out_dtype) == 0, HN_ERR_ALIGN,
            "hn_dequantize_fp4: q and s need 16-byte aligned rows, out its type's alignment");
    CHECK_DEVICE(q);
    return launched(launch_dequant_fp4(q, ldq, s, r, M, K, Kp, kind - HN_KIND_MXFP4, out, ldo, out_dtype, (cudaStream_t)stream),
                    "hn_dequantize_fp4 launch");
}

int hn_fp4_gemm(const void *qa, int64_t lda, const void *sa, const float *ra, const void *qw, int64_t ldw, const void *sw,
                const float *rw, const void *bias, int bias_dtype, void *out, int64_t ldo, int out_dtype, int64_t M, int64_t N,
                int64_t K, int kind, void *stream) {
    REQUIRE(fp4_kind(kind), HN_ERR_ARG, "hn_fp4_gemm: unknown kind %d", kind);
    REQUIRE(float_dtype(out_dtype), HN_ERR_ARG, "hn_fp4_gemm: bad out_dtype %d", out_dtype);
    REQUIRE(M >= 0 && M <= 0x7fffff00LL && N > 0 && N <= 0x7fffff00LL && K > 0 && K <= (1LL << 30) && K % 32 == 0, HN_ERR_SHAPE,
            "hn_fp4_gemm: need N > 0 and K %% 32 == 0 (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
    REQUIRE(cdiv(M, 128) * cdiv(N, 128) <= 0x7fffffffLL / 16, HN_ERR_SHAPE, "hn_fp4_gemm: too many outputs");
    REQUIRE(kind == HN_KIND_NVFP4 || (ra == nullptr && rw == nullptr), HN_ERR_ARG, "hn_fp4_gemm: row scales are for HN_KIND_NVFP4");
    REQUIRE(bias == nullptr || float_dtype(bias_dtype), HN_ERR_ARG, "hn_fp4_gemm: bad bias dtype %d", bias_dtype);
    if (M == 0) return HN_OK;
    REQUIRE(qa && sa && qw && sw && out, HN_ERR_ARG, "hn_fp4_gemm: null pointer");
    REQUIRE(lda >= K / 2 && ldw >= K / 2 && ldo >= N, HN_ERR_SHAPE, "hn_fp4_gemm: leading dimension too small");
    REQUIRE(lda < (1LL << 40) && ldw < (1LL << 40), HN_ERR_SHAPE, "hn_fp4_gemm: leading dimension too large");
    REQUIRE(al16(qa) && al16(qw) && al16(sa) && al16(sw) && lda % 16 == 0 && ldw % 16 == 0, HN_ERR_ALIGN,
            "hn_fp4_gemm: codes and scales need 16-byte aligned rows");
    REQUIRE(al4(ra) && al4(rw) && reinterpret_cast<uintptr_t>(out) % dsize(out_dtype) == 0 &&
                (bias == nullptr || reinterpret_cast<uintptr_t>(bias) % dsize(bias_dtype) == 0), HN_ERR_ALIGN,
            "hn_fp4_gemm: out, bias and row scales need their type's alignment");
    CHECK_DEVICE(qa);
    Fp4GemmArgs a;
    a.qa = qa; a.lda = lda; a.sa = sa; a.ra = ra;
    a.qw = qw; a.ldw = ldw; a.sw = sw; a.rw = rw;
    a.bias = bias; a.bias_dtype = bias_dtype; a.out = out; a.ldo = ldo; a.out_dtype = out_dtype;
    a.M = M; a.N = N; a.K = K; a.kind = kind - HN_KIND_MXFP4;
    a.sm_reserve = gemm_sm_reserve();
    const char *msg = nullptr;
    cudaError_t e = launch_fp4_gemm(a, (cudaStream_t)stream, &msg);
    if (e != cudaSuccess && msg) return fail(HN_ERR_ALIGN, "hn_fp4_gemm: %s", msg);
    return launched(e, "hn_fp4_gemm launch");
}

// what the rotations have in common; takes the weights' type out of `layout`
static int rotation_args(const char *what, const void *pos, int wide, const int64_t *freq, int64_t rot, int &layout, float factor,
                         const void *w0, const void *w1, float eps, int64_t D, int &w_wide) {
    w_wide = layout == (HN_ROPE_HALF | HN_ROPE_NORM_FP32) || layout == (HN_ROPE_INTERLEAVED | HN_ROPE_NORM_FP32);
    if (w_wide) layout &= ~HN_ROPE_NORM_FP32;
    REQUIRE(D >= 8 && D <= 256 && D % 8 == 0 && rot >= 8 && rot <= D && rot % 8 == 0, HN_ERR_SHAPE,
            "%s: need rot <= D <= 256, both multiples of 8 (rot=%lld D=%lld)", what, (long long)rot, (long long)D);
    REQUIRE(layout == HN_ROPE_HALF || layout == HN_ROPE_INTERLEAVED, HN_ERR_ARG, "%s: unknown layout %d", what, layout);
    REQUIRE(wide == 0 || wide == 1, HN_ERR_ARG, "%s: pos_wide is 0 or 1", what);
    REQUIRE(std::isfinite(factor) && std::isfinite(eps) && eps >= 0.0f, HN_ERR_ARG, "%s: factor and eps must be finite, eps >= 0", what);
    REQUIRE(freq, HN_ERR_ARG, "%s: null pointer", what);
    REQUIRE(al8(freq) && al16(w0) && al16(w1) && reinterpret_cast<uintptr_t>(pos) % (wide ? 8 : 4) == 0, HN_ERR_ALIGN,
            "%s: weights must be 16-byte aligned, positions and frequencies as their types", what);
    return HN_OK;
}

int hn_rotate(const void *x, int64_t x_bs, int64_t x_ls, int64_t x_hs, int dtype, const void *pos, int64_t p_bs, int64_t p_ls,
              int pos_wide, const int64_t *freq, int64_t rot, int layout, float factor, const void *weight, float eps, int64_t B,
              int64_t L, int64_t H, int64_t D, void *out, int64_t o_bs, int64_t o_ls, int64_t o_hs, void *stream) {
    REQUIRE(float_dtype(dtype), HN_ERR_ARG, "hn_rotate: bad dtype %d", dtype);
    REQUIRE(B >= 0 && L >= 0 && H >= 0 && B <= 0x7fffffff && L <= 0x7fffffff && H <= 65536, HN_ERR_SHAPE,
            "hn_rotate: bad shape (B=%lld L=%lld H=%lld)", (long long)B, (long long)L, (long long)H);
    int w_wide = 0;
    if (int rc = rotation_args("hn_rotate", pos, pos_wide, freq, rot, layout, factor, weight, nullptr, eps, D, w_wide)) return rc;
    if (B == 0 || L == 0 || H == 0) return HN_OK;
    REQUIRE(B * L <= (1LL << 40) / H, HN_ERR_SHAPE, "hn_rotate: too many heads");
    REQUIRE(x && pos && out, HN_ERR_ARG, "hn_rotate: null pointer");
    REQUIRE(al16(x) && al16(out) && (x_bs | x_ls | x_hs | o_bs | o_ls | o_hs) % 8 == 0, HN_ERR_ALIGN,
            "hn_rotate: x and out must be 16-byte aligned, strides multiples of 8 elements");
    REQUIRE(rows_apart(B, o_bs, L, o_ls, H, o_hs, D), HN_ERR_SHAPE, "hn_rotate: the heads of out overlap");
    CHECK_DEVICE(x);
    RotateArgs a;
    a.x = x; a.x_bs = x_bs; a.x_ls = x_ls; a.x_hs = x_hs;
    a.out = out; a.o_bs = o_bs; a.o_ls = o_ls; a.o_hs = o_hs; a.dtype = dtype;
    a.pos = pos; a.p_bs = p_bs; a.p_ls = p_ls; a.wide = pos_wide; a.w = weight; a.w_wide = w_wide;
    a.freq = freq; a.rot = (int)rot; a.layout = layout; a.factor = factor; a.eps = eps;
    a.B = (int)B; a.L = (int)L; a.H = (int)H; a.D = (int)D;
    return launched(launch_rotate(a, (cudaStream_t)stream), "hn_rotate launch");
}

int hn_cache_append_rotated(const hn_kv_cache *cache, int64_t layer, const void *q, int64_t q_bs, int64_t q_ts, int64_t q_hs,
                            int64_t H, const void *k, int64_t k_bs, int64_t k_ts, int64_t k_hs, const void *v, int64_t v_bs,
                            int64_t v_ts, int64_t v_hs, const int32_t *rows, int64_t B, int64_t n, const void *pos, int64_t p_bs,
                            int64_t p_ts, int pos_wide, const int64_t *freq, int64_t rot, int layout, float factor,
                            const void *q_weight, const void *k_weight, float eps, void *out, void *stream) {
    CacheArgs c;
    if (int rc = cache_args(cache, "hn_cache_append_rotated", c)) return rc;
    REQUIRE(layer >= 0 && layer < cache->layers, HN_ERR_SHAPE, "hn_cache_append_rotated: layer %lld of %lld", (long long)layer,
            (long long)cache->layers);
    REQUIRE(B >= 0 && n >= 0 && B <= MAX_REQUESTS && n <= 0x3fffffff && H >= 1 && H <= 65536, HN_ERR_SHAPE,
            "hn_cache_append_rotated: bad count");
    int w_wide = 0;
    if (int rc = rotation_args("hn_cache_append_rotated", pos, pos_wide, freq, rot, layout, factor, q_weight, k_weight, eps, 128, w_wide))
        return rc;
    if (B == 0 || n == 0) return HN_OK;
    REQUIRE(q && k && v && rows && out, HN_ERR_ARG, "hn_cache_append_rotated: null pointer");
    REQUIRE(al16(q) && al16(k) && al16(v) && al16(out) &&
                (q_bs | q_ts | q_hs | k_bs | k_ts | k_hs | v_bs | v_ts | v_hs) % 8 == 0, HN_ERR_ALIGN,
            "hn_cache_append_rotated: q, k, v and out need 16-byte aligned rows of 128");
    REQUIRE(cache->refused, HN_ERR_ARG, "hn_cache_append_rotated: null pointer in the cache");
    REQUIRE(cache->epoch != 0, HN_ERR_ARG, "hn_cache_append_rotated: the cache's epoch is 0");
    CHECK_DEVICE(k);
    AppendRotatedArgs a;
    a.x[0] = q; a.bs[0] = q_bs; a.ts[0] = q_ts; a.hs[0] = q_hs;
    a.x[1] = k; a.bs[1] = k_bs; a.ts[1] = k_ts; a.hs[1] = k_hs;
    a.x[2] = v; a.bs[2] = v_bs; a.ts[2] = v_ts; a.hs[2] = v_hs;
    a.out = out; a.rows = rows; a.pos = pos; a.p_bs = p_bs; a.p_ts = p_ts; a.wide = pos_wide;
    a.w[0] = q_weight; a.w[1] = k_weight; a.w_wide = w_wide;
    a.freq = freq; a.rot = (int)rot; a.layout = layout; a.factor = factor; a.eps = eps;
    a.B = (int)B; a.n = (int)n; a.H = (int)H;
    return launched(launch_append_rotated(c, (int)layer, a, (cudaStream_t)stream), "hn_cache_append_rotated launch");
}

} // extern "C"

// ---------------------------------------------------------------------------------------------------
// Sequence-parallel K/V exchange over NVLink by the copy engines (host-side only: CUDA IPC mappings, an
// asynchronous peer copy, a 32-bit flag write the GPU's front end executes after the copy - no SM involved - and a
// one-warp bounded wait for the peers' flags). No reference counterpart: the reference runs one GPU.

namespace hn {

typedef CUresult(CUDAAPI *PfnWrite32)(CUstream, CUdeviceptr, cuuint32_t, unsigned int);
typedef CUresult(CUDAAPI *PfnAddrRange)(CUdeviceptr *, size_t *, CUdeviceptr);

template <typename F> static F driver_fn(const char *name) {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion(name, &ptr, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    return reinterpret_cast<F>(ptr);
}

static int cu_fail(CUresult r, const char *what) {
    return fail(HN_ERR_CUDA, "%s failed (CUresult %d)", what, (int)r);
}

} // namespace hn

extern "C" {

int hn_ipc_export(const void *ptr, void *handle_host, int64_t *offset_host) {
    REQUIRE(ptr && handle_host && offset_host, HN_ERR_ARG, "hn_ipc_export: null pointer");
    static PfnAddrRange range = driver_fn<PfnAddrRange>("cuMemGetAddressRange");
    REQUIRE(range != nullptr, HN_ERR_CUDA, "hn_ipc_export: cuMemGetAddressRange unavailable");
    CUdeviceptr base = 0;
    size_t size = 0;
    CUresult r = range(&base, &size, reinterpret_cast<CUdeviceptr>(ptr));
    if (r != CUDA_SUCCESS) return cu_fail(r, "cuMemGetAddressRange");
    cudaIpcMemHandle_t h;
    cudaError_t e = cudaIpcGetMemHandle(&h, reinterpret_cast<void *>(base));
    if (e != cudaSuccess) return cuda_fail(e, "cudaIpcGetMemHandle");
    memcpy(handle_host, &h, sizeof(h));
    *offset_host = (int64_t)(reinterpret_cast<CUdeviceptr>(ptr) - base);
    t_last_error.clear();
    return HN_OK;
}

int hn_ipc_import(const void *handle_host, void **base_host) {
    REQUIRE(handle_host && base_host, HN_ERR_ARG, "hn_ipc_import: null pointer");
    cudaIpcMemHandle_t h;
    memcpy(&h, handle_host, sizeof(h));
    void *base = nullptr;
    cudaError_t e = cudaIpcOpenMemHandle(&base, h, cudaIpcMemLazyEnablePeerAccess);
    if (e != cudaSuccess) return cuda_fail(e, "cudaIpcOpenMemHandle");
    *base_host = base;
    t_last_error.clear();
    return HN_OK;
}

int hn_ipc_close(void *base) {
    REQUIRE(base != nullptr, HN_ERR_ARG, "hn_ipc_close: null pointer");
    cudaError_t e = cudaIpcCloseMemHandle(base);
    if (e != cudaSuccess) return cuda_fail(e, "cudaIpcCloseMemHandle");
    t_last_error.clear();
    return HN_OK;
}

int hn_peer_push(void *dst, const void *src, int64_t bytes, void *flag, uint32_t value, void *stream) {
    REQUIRE(dst && src && bytes >= 0, HN_ERR_ARG, "hn_peer_push: null pointer or negative size");
    static PfnWrite32 write32 = driver_fn<PfnWrite32>("cuStreamWriteValue32");
    REQUIRE(flag == nullptr || write32 != nullptr, HN_ERR_CUDA, "hn_peer_push: cuStreamWriteValue32 unavailable");
    StreamDevice sd(stream);
    if (sd.err != cudaSuccess) return cuda_fail(sd.err, "cudaStreamGetDevice");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (bytes > 0) {
        cudaError_t e = cudaMemcpyAsync(dst, src, (size_t)bytes, cudaMemcpyDeviceToDevice, st);
        if (e != cudaSuccess) return cuda_fail(e, "cudaMemcpyAsync (peer push)");
    }
    if (flag != nullptr) {
        // default flags: a memory fence precedes the write, so the copy above is visible before the flag
        CUresult r = write32(reinterpret_cast<CUstream>(st), reinterpret_cast<CUdeviceptr>(flag), value, 0);
        if (r != CUDA_SUCCESS) return cu_fail(r, "cuStreamWriteValue32");
    }
    t_last_error.clear();
    return HN_OK;
}

int hn_peer_push2d(void *dst, int64_t dpitch, const void *src, int64_t spitch, int64_t width, int64_t height,
                   void *flag, uint32_t value, void *stream) {
    REQUIRE(dst && src, HN_ERR_ARG, "hn_peer_push2d: null pointer");
    REQUIRE(width >= 0 && height >= 0 && dpitch >= width && spitch >= width, HN_ERR_SHAPE,
            "hn_peer_push2d: need 0 <= width <= pitches and height >= 0 (width=%lld dpitch=%lld spitch=%lld "
            "height=%lld)", (long long)width, (long long)dpitch, (long long)spitch, (long long)height);
    static PfnWrite32 write32 = driver_fn<PfnWrite32>("cuStreamWriteValue32");
    REQUIRE(flag == nullptr || write32 != nullptr, HN_ERR_CUDA, "hn_peer_push2d: cuStreamWriteValue32 unavailable");
    StreamDevice sd(stream);
    if (sd.err != cudaSuccess) return cuda_fail(sd.err, "cudaStreamGetDevice");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (width > 0 && height > 0) {
        cudaError_t e = cudaMemcpy2DAsync(dst, (size_t)dpitch, src, (size_t)spitch, (size_t)width, (size_t)height,
                                          cudaMemcpyDeviceToDevice, st);
        if (e != cudaSuccess) return cuda_fail(e, "cudaMemcpy2DAsync (peer push)");
    }
    if (flag != nullptr) {
        // default flags: a memory fence precedes the write, so the rows above are visible before the flag
        CUresult r = write32(reinterpret_cast<CUstream>(st), reinterpret_cast<CUdeviceptr>(flag), value, 0);
        if (r != CUDA_SUCCESS) return cu_fail(r, "cuStreamWriteValue32");
    }
    t_last_error.clear();
    return HN_OK;
}

int hn_wait_flags(const int32_t *flags, int64_t groups, int64_t count, int64_t group_stride, int64_t skip,
                  uint32_t value, uint32_t timeout_us, void *stream) {
    REQUIRE(flags != nullptr, HN_ERR_ARG, "hn_wait_flags: null pointer");
    REQUIRE(groups >= 0 && count >= 0 && groups <= 1024 && count <= 1024 && groups * count <= 1024, HN_ERR_SHAPE,
            "hn_wait_flags: need 0 <= groups * count <= 1024 (groups=%lld count=%lld)", (long long)groups,
            (long long)count);
    REQUIRE(group_stride >= 0 && group_stride <= (1LL << 20), HN_ERR_SHAPE, "hn_wait_flags: group_stride out of range");
    REQUIRE(timeout_us > 0 && timeout_us <= 600000000u, HN_ERR_ARG, "hn_wait_flags: timeout_us must be in (0, 6e8]");
    REQUIRE(((uintptr_t)flags % 4) == 0, HN_ERR_ALIGN, "hn_wait_flags: flags must be 4-byte aligned");
    if (groups * count == 0) return HN_OK;
    CHECK_DEVICE(flags);
    return launched(launch_wait_flags(reinterpret_cast<const uint32_t *>(flags), (int)groups, (int)count,
                                      (int)group_stride, (int)(skip < 0 || skip >= count ? -1 : skip), value,
                                      timeout_us, static_cast<cudaStream_t>(stream)),
                    "hn_wait_flags launch");
}

} // extern "C"
