// Rows into 8-bit integers with one scale each: s = max |x| / 127, code = the integer nearest x / s (half to even).
//
// A row is held in the registers of its threads between the maximum and the codes, so it is read once (beyond 4096 vectors of 16 bytes, 16384 fp32 or 32768 bf16 values, what is beyond is
// fetched again): bound by HBM (2 or 4 bytes in, one out).  y = x RN(1/s) is off
// the quotient by less than 2^-15, so rint(y) is the code unless y lies that near to a half; a vector in which one does is coded again by exact residuals:
// where x - c s of the code c = rint(y) (exact in one FMA: c has 7 bits and cancels all but the last bits of x) lies beyond s / 2, or on it with c odd,
// the neighbour is the code.  The first way takes 5 operations a value (packed products, the rounding by adding 1.5 2^23, whose low byte is the code), the
// second, for every value, took 43: 14336 x 4096 bf16 42 us (4.2 TB/s) against 72, 2047 x 14336 fp32 30 (4.9 TB/s) against 47.  What keeps bf16 from HBM's rate: a CTA's loads stop while
// it reduces and codes its row.
#include "rows.cuh"

namespace mab {
namespace quant8 {

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

// |x| of a vector, the largest; NaN where there is one.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float magnitude(uint4 r, const float*) {
    return max_nan(max_nan(fabsf(__uint_as_float(r.x)), fabsf(__uint_as_float(r.y))), max_nan(fabsf(__uint_as_float(r.z)), fabsf(__uint_as_float(r.w))));
}
__device__ __forceinline__ float magnitude(uint4 r, const uint16_t*) {
    uint32_t a, b;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(r.x & 0x7FFF7FFFu), "r"(r.y & 0x7FFF7FFFu));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(r.z & 0x7FFF7FFFu), "r"(r.w & 0x7FFF7FFFu));
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    return max_nan(__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u));
}

// The codes of a vector, a byte each.
template <typename T, int N> __device__ __forceinline__ void codes_of(uint4 r, float s, float inv, uint32_t (&w)[N / 4]) {
    constexpr float MAGIC = 12582912.0f;             // 1.5 2^23
    uint64_t x[N / 2];
    unpack_pairs(r, x, (const T*)nullptr);
    const uint64_t inv2 = pair_of(inv, inv), up = pair_of(MAGIC, MAGIC), down = pair_of(-MAGIC, -MAGIC), minus = pair_of(-1.0f, -1.0f);
    float far = 0.0f;
    uint32_t c[N];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const uint64_t y = mul2(x[i], inv2), m = add2(y, up), t = fma2(add2(m, down), minus, y);      // y - rint(y), exact
        float lo, hi;
        split(t, lo, hi);
        far = fmaxf(far, fmaxf(fabsf(lo), fabsf(hi)));
        c[2 * i] = (uint32_t)m;
        c[2 * i + 1] = (uint32_t)(m >> 32);
    }
    if (far > 0.5f - 6.103515625e-05f) {
        float v[N];
        unpack(r, v, (const T*)nullptr);
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = (uint32_t)code_of(v[i], s, inv);
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
        w[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040), __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
}

// TPR threads share a row, each holds up to HELD vectors of it.  What limits the rate is how many bytes are on their way, so the registers are kept to those of
// 1536 threads an SM where four vectors are enough.
template <typename T, int TPR, int NT, int HELD>
__global__ void __launch_bounds__(NT, HELD == 4 ? 1536 / NT : 1024 / NT) quantize_rows_kernel(Args a) {
    constexpr int N = RowGrid<T>::N;
    __shared__ float s_max[NT / 32];
    const int64_t row = (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
    const int t = threadIdx.x % TPR;
    const bool there = row < a.rows;
    const RowGrid<T> g(reinterpret_cast<const T*>(a.x) + (there ? row : 0) * a.pitch, a.cols);
    const int w0 = g.whole_from(0), w1 = g.whole_to(g.count);
    kernel_before_is_done();
    auto fetch = [&](int v) {                       // any vector; zeros outside the row
        if (v >= w0 && v < w1) return g.stream(v);
        float x[N];
        g.load_part(v, x, 0.0f);
        return pack(x, (const T*)nullptr);
    };
    uint4 held[HELD];
    float top = 0.0f;
    if (there) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) if (t + i * TPR < g.count) held[i] = fetch(t + i * TPR);
#pragma unroll
        for (int i = 0; i < HELD; ++i) if (t + i * TPR < g.count) top = max_nan(top, magnitude(held[i], (const T*)nullptr));
        for (int v = t + HELD * TPR; v < g.count; v += TPR) top = max_nan(top, magnitude(fetch(v), (const T*)nullptr));      // what the registers do not hold
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (TPR > 32) {
        if (lane_id() == 0) s_max[warp_id()] = top;
        __syncthreads();
        const int first = threadIdx.x / TPR * (TPR / 32);
#pragma unroll
        for (int w = 0; w < TPR / 32; ++w) top = max_nan(top, s_max[first + w]);
    }
    if (!there) return;
    float s = __fdiv_rn(top, 127.0f);
    if (s < 1.17549435e-38f) s = 0.0f;
    const bool finite = top < INF_F, coded = s > 0.0f && finite;               // (a NaN is not below)
    if (!finite) s = __uint_as_float(0x7FC00000u);
    if (t == 0) a.scales[row] = s;
    const float inv = coded ? __frcp_rn(s) : 0.0f;
    int8_t* out = a.codes + row * a.codes_pitch;
    const bool aligned = (reinterpret_cast<uintptr_t>(out + g.first(0)) & (N - 1)) == 0;
    auto put = [&](int v, uint4 r) {
        uint32_t w[N / 4];
#pragma unroll
        for (int i = 0; i < N / 4; ++i) w[i] = 0;
        if (coded) codes_of<T, N>(r, s, inv, w);
        const int e = g.first(v);
        if (aligned && v >= w0 && v < w1) {
            if (N == 8) *reinterpret_cast<uint2*>(out + e) = make_uint2(w[0], w[N / 4 - 1]);
            else *reinterpret_cast<uint32_t*>(out + e) = w[0];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) if (e + i >= 0 && e + i < g.n) out[e + i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
        }
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i) if (t + i * TPR < g.count) put(t + i * TPR, held[i]);
    for (int v = t + HELD * TPR; v < g.count; v += TPR) put(v, fetch(v));
}

template <typename T> int launch(const Args& a, cudaStream_t s) {
    // a warp for short rows (four rows a CTA), otherwise as many threads as hold the row
    const int64_t vectors = ceil_div64(a.cols, RowGrid<T>::N) + 1;
    if (vectors <= 32 * 4) return launch_rows(quantize_rows_kernel<T, 32, 128, 4>, "quantize_rows", ceil_div64(a.rows, 4), 128, 0, 1, s, a);
    if (vectors <= 128 * 4 + 1) return launch_rows(quantize_rows_kernel<T, 128, 128, 4>, "quantize_rows", a.rows, 128, 0, 1, s, a);
    if (vectors <= 256 * 4 + 1) return launch_rows(quantize_rows_kernel<T, 256, 256, 4>, "quantize_rows", a.rows, 256, 0, 1, s, a);
    if (vectors <= 512 * 4 + 1) return launch_rows(quantize_rows_kernel<T, 512, 512, 4>, "quantize_rows", a.rows, 512, 0, 1, s, a);
    return launch_rows(quantize_rows_kernel<T, 512, 512, 8>, "quantize_rows", a.rows, 512, 0, 1, s, a);
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
    const int64_t e = x_dtype == MAB_F32 ? 4 : 2;
    const Span in = {x, rows, cols * e, x_pitch * e}, out = {codes, rows, cols, codes_pitch}, out_scales = vector_span(scales, rows * 4);
    MAB_REQUIRE(apart(in, out) && apart(in, out_scales) && apart(out, out_scales), MAB_ERR_BAD_ARG, "mab_quantize_rows: the codes or scales overlap one another or x");
    quant8::Args a = {x, x_pitch, codes_pitch, codes, scales, rows, (int)cols};
    return x_dtype == MAB_F32 ? quant8::launch<float>(a, (cudaStream_t)stream) : quant8::launch<uint16_t>(a, (cudaStream_t)stream);
}
