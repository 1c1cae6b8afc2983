// Rows into 8-bit integers with one scale each: s = max |x| / 127, code = the integer nearest x / s (half to even).
//
// A row is held in the registers of its threads between the maximum and the codes, so it is read once: bound by HBM (2 or 4 bytes in, one
// out).  A quotient next to a half decides by its exact value: y = x RN(1/s) is off by a few units of its last place, and where the residual
// x - c s of the code c = rint(y) (exact in one FMA: c has 7 bits and cancels all but the last bits of x) lies beyond s / 2, or on it with
// c odd, the neighbour is the code.  That is 8 operations a value instead of a division's twenty.
#include "rows.cuh"

namespace mab {
namespace quant8 {

constexpr int HELD = 8;                       // vectors of 16 bytes a thread holds

struct Args {
    const void* x;
    int64_t pitch, codes_pitch;
    int8_t* codes;
    float* scales;
    int64_t rows;
    int cols;
};

// rint(x / s) of the exact quotient, for 2^-126 <= s finite, |x| <= 127 s (1 + 2^-23), inv = RN(1 / s)
__device__ __forceinline__ int code_of(float x, float s, float inv) {
    float c = rintf(__fmul_rn(x, inv));
    const float d = __fmul_rn(2.0f, __fmaf_rn(-c, s, x));      // twice the residual
    const float up = d < 0.0f ? -1.0f : 1.0f;
    const int odd = __float2int_rn(c) & 1;
    if (fabsf(d) > s || (fabsf(d) == s && odd)) c += up;
    return __float2int_rn(c);
}

// TPR threads share a row.
template <typename T, int TPR, int NT>
__global__ void __launch_bounds__(NT) quantize_rows_kernel(Args a) {
    constexpr int N = RowGrid<T>::N;
    __shared__ uint32_t s_max[NT / 32];
    const int64_t row = (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
    const int t = threadIdx.x % TPR;
    const bool there = row < a.rows;
    const RowGrid<T> g(reinterpret_cast<const T*>(a.x) + (there ? row : 0) * a.pitch, a.cols);
    // |x| bits: an infinity or a NaN is not below those of infinity
    uint32_t top = 0;
    auto see = [&](const float (&x)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    };
    uint4 held[HELD];
    if (there) {
        const int w0 = g.whole_from(0), w1 = g.whole_to(g.count);
#pragma unroll
        for (int i = 0; i < HELD; ++i) if (t + i * TPR >= w0 && t + i * TPR < w1) held[i] = g.load(t + i * TPR);
#pragma unroll
        for (int i = 0; i < HELD; ++i) if (t + i * TPR >= w0 && t + i * TPR < w1) {
            float x[N];
            unpack(held[i], x, (const T*)nullptr);
            see(x);
        }
        for (int v = t; v < g.count; v += TPR) {               // what the registers do not hold, and the partial vectors
            if (v < HELD * TPR && v >= w0 && v < w1) continue;
            float x[N];
            if (v >= w0 && v < w1) unpack(g.load(v), x, (const T*)nullptr);
            else g.load_part(v, x, 0.0f);
            see(x);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (TPR > 32) {
        if (lane_id() == 0) s_max[warp_id()] = top;
        __syncthreads();
        const int w0 = threadIdx.x / TPR * (TPR / 32);
#pragma unroll
        for (int w = 0; w < TPR / 32; ++w) top = max(top, s_max[w0 + w]);
    }
    if (!there) return;
    float s = __fdiv_rn(__uint_as_float(top), 127.0f);
    if (s < 1.17549435e-38f) s = 0.0f;
    const bool coded = s > 0.0f && top < 0x7F800000u;
    if (top >= 0x7F800000u) s = __uint_as_float(0x7FC00000u);
    if (t == 0) a.scales[row] = s;
    const float inv = coded ? __frcp_rn(s) : 0.0f;
    int8_t* out = a.codes + row * a.codes_pitch;
    auto put = [&](int v, const float (&x)[N]) {
        int c[N];
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = coded ? code_of(x[i], s, inv) : 0;
        const int e = g.first(v);
        int8_t* o = out + e;
        if (e >= 0 && e + N <= g.n && (reinterpret_cast<uintptr_t>(o) & (N - 1)) == 0) {
            uint32_t w[N / 4];
#pragma unroll
            for (int i = 0; i < N / 4; ++i)
                w[i] = (uint32_t)(c[4 * i] & 255) | (uint32_t)(c[4 * i + 1] & 255) << 8 | (uint32_t)(c[4 * i + 2] & 255) << 16 | (uint32_t)c[4 * i + 3] << 24;
            if (N == 8) *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[N / 4 - 1]);
            else *reinterpret_cast<uint32_t*>(o) = w[0];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) if (e + i >= 0 && e + i < g.n) o[i] = (int8_t)c[i];
        }
    };
    const int w0 = g.whole_from(0), w1 = g.whole_to(g.count);
#pragma unroll
    for (int i = 0; i < HELD; ++i) if (t + i * TPR >= w0 && t + i * TPR < w1) {
        float x[N];
        unpack(held[i], x, (const T*)nullptr);
        put(t + i * TPR, x);
    }
    for (int v = t; v < g.count; v += TPR) {
        if (v < HELD * TPR && v >= w0 && v < w1) continue;
        float x[N];
        if (v >= w0 && v < w1) unpack(g.load(v), x, (const T*)nullptr);
        else g.load_part(v, x, 0.0f);
        put(v, x);
    }
}

template <typename T> int launch(const Args& a, cudaStream_t s) {
    const int64_t vectors = ceil_div64(a.cols, RowGrid<T>::N) + 1;
    if (vectors <= 32 * 2) return launch_rows(quantize_rows_kernel<T, 32, 128>, "quantize_rows", ceil_div64(a.rows, 4), 128, 0, 1, s, a);
    if (vectors <= 128 * HELD) return launch_rows(quantize_rows_kernel<T, 128, 128>, "quantize_rows", a.rows, 128, 0, 1, s, a);
    return launch_rows(quantize_rows_kernel<T, 512, 512>, "quantize_rows", a.rows, 512, 0, 1, s, a);
}

}  // namespace quant8
}  // namespace mab

using namespace mab;

extern "C" int mab_quantize_rows(int64_t rows, int64_t cols, const void* x, int x_dtype, int64_t x_pitch, int8_t* codes,
                                 int64_t codes_pitch, float* scales, void* stream) {
    MAB_REQUIRE(rows >= 0 && cols >= 1, MAB_ERR_BAD_ARG, "mab_quantize_rows: rows=%lld, cols=%lld", (long long)rows, (long long)cols);
    MAB_REQUIRE(x_dtype == MAB_F32 || x_dtype == MAB_BF16, MAB_ERR_UNSUPPORTED, "mab_quantize_rows: element type %d", x_dtype);
    MAB_REQUIRE(rows <= INT32_MAX && cols <= (1 << 30), MAB_ERR_LIMIT, "mab_quantize_rows: rows=%lld, cols=%lld", (long long)rows, (long long)cols);
    if (rows == 0) return MAB_OK;
    MAB_REQUIRE(x && codes && scales, MAB_ERR_BAD_ARG, "mab_quantize_rows: null pointer");
    MAB_REQUIRE(x_pitch >= cols && codes_pitch >= cols, MAB_ERR_BAD_ARG, "mab_quantize_rows: rows of %lld values lie %lld and %lld apart", (long long)cols,
                (long long)x_pitch, (long long)codes_pitch);
    MAB_REQUIRE(aligned_to(x, x_dtype == MAB_F32 ? 4 : 2) && aligned_to(scales, 4), MAB_ERR_BAD_ARG, "mab_quantize_rows: misaligned buffer");
    quant8::Args a = {x, x_pitch, codes_pitch, codes, scales, rows, (int)cols};
    return x_dtype == MAB_F32 ? quant8::launch<float>(a, (cudaStream_t)stream) : quant8::launch<uint16_t>(a, (cudaStream_t)stream);
}
