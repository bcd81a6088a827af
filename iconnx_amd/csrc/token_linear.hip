// Int8 matrix product with a scale for each token and each output channel:
//   s_m = max(max_k |x_mk| / 127, 2^-126),  q_mk = rne(x_mk / s_m)
//   y_mn = (sum_k q_mk w_kn) (s_m w_scale_n) + bias_n
// A token whose values are not all finite has the scale NaN and the codes 0, so that its outputs are
// NaN and nobody else's are.
//
// Weights are packed once, transposed to [N, Kp] with Kp = K rounded up to 128 and zeros past K;
// quantized tokens that this library makes for itself have rows of Kp bytes too, so that the
// product kernels never see a ragged K.
#include "elem.hpp"
#include "internal.hpp"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr size_t kAlignK = 128;

inline size_t padded(size_t K) { return icx::align_up(K, kAlignK); }

// ---- weights --------------------------------------------------------------------------------
// 64 x 64 bytes through LDS: rows of b in, rows of the transpose out, zeros past K.
__global__ void __launch_bounds__(kThreads) token_weight_pack_kernel(const int8_t* b, int64_t K, int64_t N, int64_t Kp,
                                                                     int8_t* out) {
    __shared__ int8_t tile[64][65];
    const int64_t k0 = (int64_t)blockIdx.x * 64, n0 = (int64_t)blockIdx.y * 64;
    const int c = threadIdx.x & 63;
    for (int r = threadIdx.x >> 6; r < 64; r += 4)
        tile[r][c] = k0 + r < K && n0 + c < N ? b[(k0 + r) * N + n0 + c] : (int8_t)0;
    __syncthreads();
    for (int r = threadIdx.x >> 6; r < 64; r += 4)
        if (n0 + r < N) out[(n0 + r) * Kp + k0 + c] = tile[c][r];
}

// ---- quantization of tokens -------------------------------------------------------------------
struct TokenScale {
    float s, inv;
};
// From the bits of the largest magnitude of the row (NaN above infinity above the rest).
__device__ __forceinline__ TokenScale token_scale(uint32_t top) {
    if (top >= 0x7f800000u) return {__builtin_nanf(""), 0.0f};
    const float s = fmaxf(__uint_as_float(top) / 127.0f, 0x1p-126f);
    return {s, 1.0f / s};
}

// rne(x / s) of the exact quotient.  x inv is within 2e-5 of it (|x / s| <= 127, two roundings), so
// away from the halves both round alike; near one the quotient is taken in 64 bits, where it cannot
// round onto a half that it does not reach (a difference from a half is at least 2^-25 of it).
__device__ __forceinline__ int quant1(float x, const TokenScale& t) {
    const float v = x * t.inv;
    float r = rintf(v);
    if (fabsf(v - r) > 0.4999f) r = (float)rint((double)x / (double)t.s);
    return (int)r;
}

__device__ __forceinline__ uint32_t quant4(const float* x, const TokenScale& t) {
    return (uint32_t)(quant1(x[0], t) & 255) | (uint32_t)(quant1(x[1], t) & 255) << 8 | (uint32_t)(quant1(x[2], t) & 255) << 16 |
           (uint32_t)quant1(x[3], t) << 24;
}

// A wave a row.  x's rows start anywhere; q's rows have ldq bytes and are written 8 at a time where
// that is aligned (VEC), zeros from K to `fill`.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) token_quantize_kernel(const T* x, int64_t M, int K, int64_t ldx, int8_t* q, int64_t ldq,
                                                                  int fill, float* scale) {
    const int64_t m = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (m >= M) return;
    const T* row = x + m * ldx;
    uint32_t top = 0;
    const int whole = K & ~7;
    for (int k = lane * 8; k < whole; k += 512) {
        float v[8];
        icx::load_f32(row + k, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    }
    if (whole + lane < K) top = max(top, __float_as_uint((float)row[whole + lane]) & 0x7fffffffu);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
    const TokenScale t = token_scale(top);
    if (lane == 0) scale[m] = t.s;
    int8_t* out = q + m * ldq;
    const bool bad = !(t.s == t.s);
    for (int k = lane * 8; k < (VEC ? fill : K); k += 512) {
        float v[8];
        if (k + 8 <= K) icx::load_f32(row + k, v);
        else
            for (int e = 0; e < 8; ++e) v[e] = k + e < K ? (float)row[k + e] : 0.0f;
        uint2 w = make_uint2(0u, 0u);
        if (!bad) w = make_uint2(quant4(v, t), quant4(v + 4, t));
        if (VEC) *reinterpret_cast<uint2*>(out + k) = w;
        else
            for (int e = 0; e < 8 && k + e < K; ++e) out[k + e] = (int8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
    }
}

// ---- the product --------------------------------------------------------------------------------
struct ProductArgs {
    const int8_t* q;  // [M, lda], whole 128-byte steps of K in place
    int64_t lda;
    const float* xs;
    const int8_t* w;  // [N, Kp]
    const float* ws;
    const float* bias;
    void* y;
    int64_t ldy;
    int M, N, Kp;
    int tiles_m, tiles_n;
};

__device__ __forceinline__ float finish(int acc, float xs, float ws, float bias) { return (float)acc * (xs * ws) + bias; }

// 16 tokens by 16 channels a block, K split over its waves (integers: the same sum in any order).
template <int W, typename T>
__global__ void __launch_bounds__(64 * W) token_product_small_kernel(ProductArgs g) {
    __shared__ v4i part[W][64];
    const int lane = threadIdx.x & 63, lr = lane & 15, j = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = (int)(blockIdx.x / g.tiles_m) * 16, m0 = (int)(blockIdx.x % g.tiles_m) * 16;
    const int8_t* a = g.q + (int64_t)min(m0 + lr, g.M - 1) * g.lda + 16 * j;
    const int8_t* b = g.w + (int64_t)min(n0 + lr, g.N - 1) * g.Kp + 16 * j;
    v4i acc = {0, 0, 0, 0};
    for (int k = wid * 64; k < g.Kp; k += 64 * W)
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const v4i*>(a + k), *reinterpret_cast<const v4i*>(b + k), acc, 0,
                                                    0, 0);
    part[wid][lane] = acc;
    __syncthreads();
    if (wid) return;
#pragma unroll
    for (int w = 1; w < W; ++w) acc += part[w][lane];
    const int n = n0 + lr;
    if (n >= g.N) return;
    const float ws = g.ws[n], bias = g.bias ? g.bias[n] : 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int m = m0 + 4 * j + r;
        if (m < g.M) reinterpret_cast<T*>(g.y)[(int64_t)m * g.ldy + n] = (T)finish(acc[r], g.xs[m], ws, bias);
    }
}

// ---- large products: 256 x 256 tiles -------------------------------------------------------------
// Eight waves, each 128 tokens by 64 channels, K in steps of 128 bytes; both operands' steps reach
// LDS by global_load_lds_dwordx4 (16 bytes a lane, no registers), two steps of 64 KB in LDS.  The
// channels are the rows of the matrix instruction and the tokens its columns, so that a lane's four
// result registers are four channels of one token; which channels a row is stands free, and row i
// of tile t is channel 16 (i / 4) + 4 t + i % 4 of the wave's 64, which gives a lane 16 consecutive
// ones over its four tiles: y is stored 16 bytes a lane from the registers, whole 128-byte lines
// a wave, with no staging.
//
// The two waves of a SIMD (w and w + 4) run half a phase apart, one reading its fragments while the
// other multiplies: every phase is a part of reads and one of 16 matrix instructions with a barrier after
// each, and waves 4 to 7 wait at one barrier more before their first phase.  A step is four phases
// (halves of the wave's tokens by halves of its channels).  The copies of step t + 1 go into the buffer
// that step t - 1 was read from: its last reads (phase 2 of the later waves) are over one barrier before
// the earlier waves' phase 0 of step t, where the first copies are issued; every wave waits for its own
// copies in phase 3, one barrier before anyone reads them.  16384 x 4096 x 4096: 228 us (2.41 POP/s; the
// 16 x 16 tiles below 3600 us).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void wait_reads() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// 16 bytes a lane from base + offset (a lane's own) to LDS at lds + 16 lane.
__device__ __forceinline__ void copy_to_lds(const void* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// The 16-byte chunk c of a row stands at c ^ key(row) of it: the 16 rows that a fragment read takes
// together then lie in 16 different groups of banks (two rows of 128 bytes span the banks once).
__device__ __forceinline__ int token_key(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int channel_key(int row) { return ((row >> 1) & 1) | ((row >> 4) & 3) << 1; }

// Tiles in runs of one XCD (block i runs on XCD i % 8), 8 rows of tiles deep, so that the tiles that
// run together share their operands in its L2.
__device__ __forceinline__ void tile_of(const ProductArgs& g, int& tm, int& tn) {
    int i = blockIdx.x;
    const int n = gridDim.x, each = n >> 3, more = n & 7, x = i & 7;
    i = x * each + min(x, more) + (i >> 3);
    const int deep = 8 * g.tiles_n;
    const int first = i / deep * 8, rows = min(8, g.tiles_m - first);
    tm = first + i % deep % rows;
    tn = i % deep / rows;
}

constexpr int kBig = 256, kStep = 128;

// 16 channels of one token from n on.
template <typename T>
__device__ __forceinline__ void store16(T* row, int n, int N, bool wide, const float (&v)[16]) {
    if (wide && n + 16 <= N) {
        typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) {
            vec w;
#pragma unroll
            for (int e = 0; e < 16 / (int)sizeof(T); ++e) w[e] = (T)v[i * (16 / sizeof(T)) + e];
            *reinterpret_cast<vec*>(row + n + i * (16 / sizeof(T))) = w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (n + e < N) row[n + e] = (T)v[e];
    }
}

template <typename T>
__global__ void __launch_bounds__(512, 2) token_product_big_kernel(ProductArgs g) {
    __shared__ __attribute__((aligned(1024))) int8_t smem[2][2 * kBig * kStep];
    int tm, tn;
    tile_of(g, tm, tn);
    const int m0 = tm * kBig, n0 = tn * kBig;
    const int lane = threadIdx.x & 63, lr = lane & 15, j = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wid >> 2, wn = wid & 3;

    // copies: 8 rows an instruction, this wave rows 32 wid .. + 31 of either operand
    const int8_t* qa = g.q + (int64_t)m0 * g.lda;
    const int8_t* wa = g.w + (int64_t)n0 * g.Kp;
    uint32_t oq[4], ow[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = wid * 32 + i * 8 + (lane >> 3);
        oq[i] = (uint32_t)((int64_t)min(row, g.M - 1 - m0) * g.lda + 16 * ((lane & 7) ^ token_key(row)));
        ow[i] = (uint32_t)((int64_t)min(row, g.N - 1 - n0) * g.Kp + 16 * ((lane & 7) ^ channel_key(row)));
    }
    const uint32_t lq = lds_address(smem) + wid * 32 * kStep, lw = lq + kBig * kStep;
    auto copy_q = [&](int buf, int kt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) copy_to_lds(qa + kt * kStep, oq[i], lq + buf * (2 * kBig * kStep) + i * 8 * kStep);
    };
    auto copy_w = [&](int buf, int kt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) copy_to_lds(wa + kt * kStep, ow[i], lw + buf * (2 * kBig * kStep) + i * 8 * kStep);
    };
    v4i acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[i][t] = v4i{0, 0, 0, 0};
    v4i fq[4][2], fw[4][2];
    auto read_q = [&](int buf, int half) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = wm * 128 + half * 64 + i * 16 + lr;
#pragma unroll
            for (int k = 0; k < 2; ++k)
                fq[i][k] = *reinterpret_cast<const v4i*>(&smem[buf][row * kStep + 16 * ((4 * k + j) ^ token_key(row))]);
        }
    };
    auto read_w = [&](int buf, int half) {
#pragma unroll
        for (int t = 2 * half; t < 2 * half + 2; ++t) {
            const int row = wn * 64 + (lr >> 2) * 16 + t * 4 + (lr & 3);
#pragma unroll
            for (int k = 0; k < 2; ++k)
                fw[t][k] = *reinterpret_cast<const v4i*>(&smem[buf][kBig * kStep + row * kStep + 16 * ((4 * k + j) ^ channel_key(row))]);
        }
    };
    auto multiply = [&](int hq, int hw) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 2 * hw; t < 2 * hw + 2; ++t)
                    acc[4 * hq + i][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[t][k], fq[i][k], acc[4 * hq + i][t], 0, 0, 0);
        __builtin_amdgcn_s_setprio(0);
    };

    const int KT = g.Kp / kStep;
    copy_q(0, 0);
    copy_w(0, 0);
    wait_copies();
    barrier();
    if (wm) barrier();
    for (int kt = 0; kt < KT; ++kt) {
        const int cur = kt & 1;
        const int next = min(kt + 1, KT - 1);  // the last step again: into the buffer nobody reads any more
        read_w(cur, 0);
        read_q(cur, 0);
        copy_q(cur ^ 1, next);
        wait_reads();
        barrier();
        multiply(0, 0);
        barrier();
        read_w(cur, 1);
        copy_w(cur ^ 1, next);
        wait_reads();
        barrier();
        multiply(0, 1);
        barrier();
        read_q(cur, 1);
        wait_reads();
        barrier();
        multiply(1, 0);
        barrier();
        wait_copies();
        barrier();
        multiply(1, 1);
        barrier();
    }
    if (!wm) barrier();

    const int n = n0 + wn * 64 + 16 * j;
    float ws[16], bias[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int c = min(n + e, g.N - 1);
        ws[e] = g.ws[c];
        bias[e] = g.bias ? g.bias[c] : 0.0f;
    }
    const bool wide = (g.ldy * sizeof(T)) % 16 == 0 && (reinterpret_cast<uintptr_t>(g.y) & 15) == 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int m = m0 + wm * 128 + i * 16 + lr;
        if (m >= g.M) continue;
        const float xs = g.xs[m];
        float v[16];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[4 * t + r] = finish(acc[i][t][r], xs, ws[4 * t + r], bias[4 * t + r]);
        store16(reinterpret_cast<T*>(g.y) + (int64_t)m * g.ldy, n, g.N, wide, v);
    }
}

// Rows of q that are not whole steps of K (a caller's own): copied with zeros behind them.
__global__ void __launch_bounds__(kThreads) token_pad_kernel(const int8_t* q, int64_t ld, int K, int Kp, int8_t* out) {
    const int64_t m = blockIdx.x;
    for (int k = threadIdx.x; k < Kp; k += kThreads) out[m * Kp + k] = k < K ? q[m * ld + k] : (int8_t)0;
}

int quantize(hipStream_t s, const void* x, int dtype, size_t M, size_t K, int64_t ldx, int8_t* q, size_t ldq, size_t fill,
             float* scale) {
    const bool vec = ldq % 8 == 0 && fill % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
    const unsigned blocks = (unsigned)icx::cdiv(M, kThreads / 64);
    return icx::with_float_type(dtype, [&](auto* t) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        if (vec) token_quantize_kernel<T, true><<<blocks, kThreads, 0, s>>>((const T*)x, M, (int)K, ldx, q, ldq, (int)fill, scale);
        else token_quantize_kernel<T, false><<<blocks, kThreads, 0, s>>>((const T*)x, M, (int)K, ldx, q, ldq, (int)fill, scale);
        ICX_LAUNCH_CHECK("token_quantize_kernel");
        return ICX_OK;
    });
}

// q [M, Kp] and, behind it, the scales (Int8 tokens: room for rows that have to be padded).
struct Workspace {
    size_t scale_off, total;
};
Workspace workspace(size_t M, size_t K, int x_dtype) {
    const size_t q = icx::align_up(M * padded(K), 256);
    return {q, q + (x_dtype == ICX_I8 ? 0 : 4 * M)};
}

// The sums stay within 32 bits: |w|, |q| <= 128.
constexpr size_t kMaxK = 131071;

int check_sizes(size_t M, size_t K, size_t N, const char* who) {
    if (K < 1 || K > kMaxK) ICX_FAIL(ICX_ERR_SHAPE, "%s: K = %zu (must be 1 to %zu)", who, K, kMaxK);
    if (M > 0x3fffffff || N > 0x3fffffff) ICX_FAIL(ICX_ERR_SHAPE, "%s: M = %zu and N = %zu must be below 2^30", who, M, N);
    return ICX_OK;
}

}  // namespace

extern "C" size_t icx_token_weight_bytes(size_t K, size_t N) { return padded(K) * N; }

extern "C" int icx_pack_token_weight(icx_stream_t stream, const int8_t* b, size_t K, size_t N, int8_t* packed) {
    icx::clear_error();
    const char* who = "PackTokenWeight";
    int rc = check_sizes(0, K, N, who);
    if (rc) return rc;
    if (N == 0) return ICX_OK;
    if (!b || !packed) ICX_FAIL(ICX_ERR_INVALID_ARG, "%s: null weight", who);
    if (N > (size_t)65535 * 64) ICX_FAIL(ICX_ERR_UNSUPPORTED, "%s: N = %zu", who, N);
    const dim3 grid((unsigned)(padded(K) / 64), (unsigned)icx::cdiv(N, 64));
    token_weight_pack_kernel<<<grid, kThreads, 0, (hipStream_t)stream>>>(b, K, N, padded(K), packed);
    ICX_LAUNCH_CHECK("token_weight_pack_kernel");
    return ICX_OK;
}

extern "C" int icx_quantize_tokens(icx_stream_t stream, const void* x, int x_dtype, size_t M, size_t K, int64_t x_stride, int8_t* q,
                                   float* scale) {
    icx::clear_error();
    const char* who = "QuantizeTokens";
    int rc = check_sizes(M, K, 0, who);
    if (rc) return rc;
    if (!icx::is_float_kind(x_dtype))
        ICX_FAIL(ICX_ERR_DTYPE, "%s: dtype %d unsupported (must be Float32, Float16 or BFloat16)", who, x_dtype);
    if (M == 0) return ICX_OK;
    if (!x || !q || !scale) ICX_FAIL(ICX_ERR_INVALID_ARG, "%s: null x, q or scale", who);
    return quantize((hipStream_t)stream, x, x_dtype, M, K, x_stride, q, K, K, scale);
}

extern "C" size_t icx_token_qlinear_workspace_size(size_t M, size_t K, size_t N, int x_dtype) {
    (void)N;
    return workspace(M, K, x_dtype).total;
}

extern "C" int icx_token_qlinear(icx_stream_t stream, const void* x, int x_dtype, int64_t x_stride, const float* x_scale, size_t M,
                                 size_t K, size_t N, const int8_t* packed, const float* w_scale, const float* bias, void* y,
                                 int y_dtype, int64_t y_stride, void* ws, size_t ws_bytes) {
    icx::clear_error();
    const char* who = "TokenQLinear";
    int rc = check_sizes(M, K, N, who);
    if (rc) return rc;
    const bool own = x_dtype != ICX_I8;
    if (own && !icx::is_float_kind(x_dtype))
        ICX_FAIL(ICX_ERR_DTYPE, "%s: x dtype %d unsupported (must be Int8, Float32, Float16 or BFloat16)", who, x_dtype);
    if (!icx::is_float_kind(y_dtype))
        ICX_FAIL(ICX_ERR_DTYPE, "%s: y dtype %d unsupported (must be Float32, Float16 or BFloat16)", who, y_dtype);
    if (own == (x_scale != nullptr))
        ICX_FAIL(ICX_ERR_INVALID_ARG, "%s: Int8 tokens come with their scales, others without (x dtype %d, scales %s)", who, x_dtype,
                 x_scale ? "given" : "missing");
    if (M == 0 || N == 0) return ICX_OK;
    if (!x || !packed || !w_scale || !y) ICX_FAIL(ICX_ERR_INVALID_ARG, "%s: null x, weight, scale or y", who);
    if (!icx::aligned16(packed)) ICX_FAIL(ICX_ERR_INVALID_ARG, "%s: the packed weight must be 16-byte aligned", who);
    const Workspace L = workspace(M, K, x_dtype);
    const bool pad = !own && (K % kAlignK || x_stride % 16 || !icx::aligned16(x));
    if ((own || pad) && (!ws || ws_bytes < L.total))
        ICX_FAIL(ICX_ERR_WORKSPACE, "%s: workspace of %zu bytes needed (got %zu)", who, L.total, ws_bytes);
    const hipStream_t s = (hipStream_t)stream;
    ProductArgs g{};
    g.q = (const int8_t*)x;
    g.lda = x_stride;
    g.xs = x_scale;
    if (own) {
        float* sc = reinterpret_cast<float*>((char*)ws + L.scale_off);
        rc = quantize(s, x, x_dtype, M, K, x_stride, (int8_t*)ws, padded(K), padded(K), sc);
        if (rc) return rc;
        g.q = (const int8_t*)ws;
        g.lda = (int64_t)padded(K);
        g.xs = sc;
    } else if (pad) {
        token_pad_kernel<<<(unsigned)M, kThreads, 0, s>>>((const int8_t*)x, x_stride, (int)K, (int)padded(K), (int8_t*)ws);
        ICX_LAUNCH_CHECK("token_pad_kernel");
        g.q = (const int8_t*)ws;
        g.lda = (int64_t)padded(K);
    }
    g.w = packed;
    g.ws = w_scale;
    g.bias = bias;
    g.y = y;
    g.ldy = y_stride;
    g.M = (int)M;
    g.N = (int)N;
    g.Kp = (int)padded(K);
    const bool big = M >= 1024 && icx::cdiv(M, kBig) * icx::cdiv(N, kBig) >= 64;
    const size_t tile = big ? kBig : 16;
    g.tiles_m = (int)icx::cdiv(M, tile);
    g.tiles_n = (int)icx::cdiv(N, tile);
    if ((uint64_t)g.tiles_m * g.tiles_n * 256 > 0xffffffffull)
        ICX_FAIL(ICX_ERR_UNSUPPORTED, "%s: %zu x %zu outputs are too many for a launch", who, M, N);
    const unsigned blocks = (unsigned)(g.tiles_m * g.tiles_n);
    return icx::with_float_type(y_dtype, [&](auto* t) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        if (big) {
            token_product_big_kernel<T><<<blocks, 512, 0, s>>>(g);
            ICX_LAUNCH_CHECK("token_product_big_kernel");
            return ICX_OK;
        }
        token_product_small_kernel<4, T><<<blocks, 256, 0, s>>>(g);
        ICX_LAUNCH_CHECK("token_product_small_kernel");
        return ICX_OK;
    });
}
