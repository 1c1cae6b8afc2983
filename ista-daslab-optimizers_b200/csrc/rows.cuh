// Rows of a dense matrix (logits, activations) read 16 bytes a lane, wherever a row starts, and what the kernels that take a cluster
// of CTAs per row share.
#pragma once
#include "common.cuh"
#include "fused.cuh"

namespace mab {

// A row of n values as a grid of 16-byte vectors: vector v holds the elements [v N - lead, v N - lead + N).  The first and the last one
// can be partial; no load reaches outside the row.
template <typename T> struct RowGrid {
    static constexpr int N = 16 / (int)sizeof(T);
    const T* p;
    int n, lead, count;                      // elements, elements of vector 0 before the row, vectors
    __device__ __forceinline__ RowGrid(const T* row, int elements) : p(row), n(elements) {
        lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
        count = (elements + lead + N - 1) / N;
    }
    __device__ __forceinline__ int first(int v) const { return v * N - lead; }
    __device__ __forceinline__ bool whole(int v) const { return first(v) >= 0 && first(v) + N <= n; }
    // the whole vectors among [v0, v1)
    __device__ __forceinline__ int whole_from(int v0) const { return v0 == 0 && lead ? 1 : v0; }
    __device__ __forceinline__ int whole_to(int v1) const { return v1 == count && (n + lead) % N ? v1 - 1 : v1; }
    __device__ __forceinline__ uint4 load(int v) const { return *reinterpret_cast<const uint4*>(p + first(v)); }
    // The same for a vector of a stream, which nobody reads again soon: what is on its way takes no line of the first cache from the rest (topk_logits of 2048 rows of 128256
    // bf16 132 us with `load`, 122 so).
    __device__ __forceinline__ uint4 stream(int v) const {
        uint4 r;
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p + first(v)) : "memory");
        return r;
    }
    // a partial vector, by elements; what lies outside the row reads as `none`
    __device__ __forceinline__ void load_part(int v, float (&x)[N], float none) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = first(v) + i;
            x[i] = e >= 0 && e < n ? Elem<T>::load(p, e) : none;
        }
    }
};

__device__ __forceinline__ void unpack(uint4 r, float (&x)[4], const float*) {
    x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
}
__device__ __forceinline__ void unpack(uint4 r, float (&x)[8], const uint16_t*) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint4 pack(const float (&x)[4], const float*) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
__device__ __forceinline__ uint4 pack(const float (&x)[8], const uint16_t*) {
    return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}

// Pairs of floats in 64 bits, for the packed instructions.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void split(uint64_t p, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void unpack_pairs(uint4 r, uint64_t (&x)[2], const float*) {
    x[0] = (uint64_t)r.y << 32 | r.x; x[1] = (uint64_t)r.w << 32 | r.z;
}
__device__ __forceinline__ void unpack_pairs(uint4 r, uint64_t (&x)[4], const uint16_t*) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (uint64_t)(w[i] & 0xFFFF0000u) << 32 | (uint64_t)(w[i] << 16);
}
// Largest of a vector's values that are not NaN (NaN where there is none).
__device__ __forceinline__ float vector_max(uint4 r, const float*) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
}
__device__ __forceinline__ float vector_max(uint4 r, const uint16_t*) {
    uint32_t a, b;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(r.x), "r"(r.y));
    asm("max.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(r.z), "r"(r.w));
    asm("max.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u));
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float INF_F = __builtin_huge_valf();
constexpr uint32_t KEY_NEG_INF = 0x007FFFFFu;       // ord_key(-inf); every number lies above it
// Order key of a value with NaN (0) below -inf and one key for the two zeros.
__device__ __forceinline__ uint32_t row_key(float x) { return x == x ? ord_key(x + 0.0f) : 0u; }

// ----------------------------------------------------------------------------- clusters of CTAs, one per row
// (every thread of every CTA, warps whole: the unaligned form costs microseconds where a warp comes to it in pieces)
__device__ __forceinline__ void cluster_arrive_wait() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// The same in two halves.  Between the beginning of a kernel and the first access to another CTA's shared memory: that CTA has begun then.
__device__ __forceinline__ void cluster_arrive() { __syncwarp(); asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { __syncwarp(); asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// Address of `p` (in this CTA's shared memory) in that of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(const void* p, int rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ double cluster_load_f64(const double* p, int rank) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(cluster_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_load_u32(const void* p, int rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ int4 cluster_load_int4(const void* p, int rank) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(cluster_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_store_u32(void* p, int rank, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void cluster_store_u64(void* p, int rank, unsigned long long v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_addr(p, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ void cluster_store_f64(void* p, int rank, double v) {
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(cluster_addr(p, rank)), "d"(v) : "memory");
}

// Kernels that are launched by `launch_rows` begin while the one before them in the stream ends (programmatic launches): what a kernel does before this call
// touches no global memory but its parameters, and every thread of every CTA makes it, since the completion of one is what the next relies on.  Its own successor may be
// launched from here on.  What is saved is the gap between two kernels: us a call in a row of calls, without and so, when it was brought in: topk_logits of 59 rows of 1363 8.2 / 6.7, int8_matmul of
// 41 x 1000 x 512 8.2 / 6.2, distill_step of 8 rows of 8000 8.2 / 6.5, 16 x 4096 x 4096 10.2 / 6.9.  A kernel that takes tensor memory makes this call behind the barrier
// that follows the allocation.
__device__ __forceinline__ void kernel_before_is_done() {
    wait_for_kernel_before();
    allow_next_kernel(0x7FFFFFFF);
}

// Rows in memory, sizes in bytes: what a call writes has to lie apart from what it reads.  Rows of both may lie between one another (a record's fields), at one distance.
struct Span {
    const void* p;
    int64_t rows, width, pitch;
};
static inline bool apart(const Span& a, const Span& b) {
    if (a.p == nullptr || b.p == nullptr || a.rows == 0 || b.rows == 0) return true;
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a.p), a1 = a0 + (a.rows - 1) * a.pitch + a.width;
    const uintptr_t b0 = reinterpret_cast<uintptr_t>(b.p), b1 = b0 + (b.rows - 1) * b.pitch + b.width;
    if (a1 <= b0 || b1 <= a0) return true;
    if ((a.rows == 1 && b.rows == 1) || (a.rows > 1 && b.rows > 1 && a.pitch != b.pitch)) return false;
    const int64_t pitch = a.rows > 1 ? a.pitch : b.pitch;
    const int64_t ahead = ((int64_t)(b0 - a0) % pitch + pitch) % pitch;            // where b's rows begin, from the beginnings of a's
    return ahead >= a.width && ahead + b.width <= pitch;
}
static inline Span vector_span(const void* p, int64_t bytes) { return {p, 1, bytes, bytes}; }

// Launches `kernel` with clusters of `cluster` CTAs (1: without) and counts it.  (Above 48 KB with the kernel's own static memory, a few KB, the size has to be allowed.)
template <typename... P, typename... A>
static int launch_rows(void (*kernel)(P...), const char* what, int64_t ctas, int threads, size_t smem, int cluster, cudaStream_t s, A... args) {
    if (smem > 32 * 1024)
        if (int rc = allow_shared_memory(reinterpret_cast<const void*>(kernel))) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    if (e != cudaSuccess) return cuda_fail(e, what);
    count_launch();
    return MAB_OK;
}

}  // namespace mab
