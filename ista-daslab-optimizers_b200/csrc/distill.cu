// Distillation from a teacher's top logits: per row a list of k (index, logit) pairs and, where the teacher gave it, the logarithm of the
// mass of everything else (`rest`), against the student's logits z.  With t_j = value_j / tau, y_v = z_v / tau,
//
//   Lp = log(sum_j exp t_j + exp rest),  p_j = exp(t_j - Lp),  p_t = exp(rest - Lp),  P = sum_j p_j + p_t  (1, or 0 where there is nothing)
//   L = log sum_v exp y_v,  L_t = log sum_{v not in the list} exp y_v,  q_v = exp(y_v - L),  q_t = exp(L_t - L)
//   loss = sum_j p_j (log p_j - log q_j) + p_t (log p_t - log q_t)
//   tau dloss/dz_v = P q_v - sum_{j: index_j = v} p_j              for v in the list
//                  = exp(y_v - L_t) (P q_t - p_t)                  elsewhere
//
// One pass over a row with a running maximum and sum, in which a bitmap in shared memory leaves out the positions of the list: the
// sum over the others is their own, not a difference of two large ones.  The k terms of the list are in 64 bits: near the optimum the loss is what is
// left of a difference, and there an error of S_t only enters with the factor q_t - p_t as long as the terms that share it are exact.
//
// A row belongs to a cluster of one to eight CTAs (few rows: more CTAs a row), which exchange six numbers through distributed shared
// memory in rank order: results do not depend on timing.
#include "rows.cuh"

namespace mab {
namespace distill {

constexpr int NT = 512, WARPS = NT / 32;
constexpr int MAX_K = 1024, PER_THREAD = MAX_K / NT;
constexpr int UNROLL = 4;                          // vectors of 16 bytes a thread has in flight
enum Mode { LOSS, STEP };

struct Args {
    const void* logits;
    int64_t pitch;
    const int32_t* indices;
    const void* values;
    int values_bf16;
    const float* rest;
    const float* weights;
    double tau;
    float scale;                                   // log2(e) / tau
    float* loss;
    float2* stats;                                 // per row: reference, factor of the positions outside the list (LOSS)
    float* list_grad;                              // [rows, k] tau dloss/dz at the list's positions (LOSS)
    void* grad;                                    // STEP, GRAD
    int64_t grad_pitch;
    const float* grad_loss;                        // GRAD: [rows], `grad_loss_stride` apart
    int64_t grad_loss_stride;
    int vocab, k, cluster;
};

struct Shared {
    double red[WARPS][3];
    double out[3];                                 // sums over the block
    double part[5];                                // this CTA's part, read by the cluster: reference, S_t, m_k, S_k, B
    double stat[4];                                // Lp, 1 / Sp, L, P
    float fmax[WARPS][2], fsum[WARPS];
    float ref, off;
    int dup;
};

__device__ __forceinline__ double list_value(const Args& a, int64_t at) {
    return a.values_bf16 ? (double)bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(a.values)[at]) : (double)reinterpret_cast<const float*>(a.values)[at];
}

// Sums of three doubles over the block, in every thread.
__device__ __forceinline__ void block_sum(Shared& sh, double& x, double& y, double& z) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
        z += __shfl_xor_sync(0xffffffffu, z, o);
    }
    if (lane_id() == 0) { sh.red[warp_id()][0] = x; sh.red[warp_id()][1] = y; sh.red[warp_id()][2] = z; }
    __syncthreads();
    x = y = z = 0.0;
    for (int w = 0; w < WARPS; ++w) { x += sh.red[w][0]; y += sh.red[w][1]; z += sh.red[w][2]; }
}

// Writes factor * exp2((z - ref) scale) over the vectors [v0, v1) of the row.
template <typename T>
__device__ __forceinline__ void write_outside(const RowGrid<T>& g, int v0, int v1, T* out, float ref, float scale, float factor) {
    constexpr int N = RowGrid<T>::N;
    const bool same = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(g.p)) & 15) == 0;
    auto put = [&](int v, float (&x)[N], bool vector) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = factor * ex2((x[i] - ref) * scale);
        if (vector) *reinterpret_cast<uint4*>(out + g.first(v)) = pack(x, (const T*)nullptr);
        else
#pragma unroll
            for (int i = 0; i < N; ++i) if (g.first(v) + i >= 0 && g.first(v) + i < g.n) Elem<T>::store(out, g.first(v) + i, x[i]);
    };
    const int w0 = g.whole_from(v0), w1 = g.whole_to(v1);
    int v = w0 + threadIdx.x;
    for (; v + (UNROLL - 1) * NT < w1; v += UNROLL * NT) {
        uint4 r[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) r[u] = g.load(v + u * NT);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) { float x[N]; unpack(r[u], x, (const T*)nullptr); put(v + u * NT, x, same); }
    }
    for (; v < w1; v += NT) { float x[N]; unpack(g.load(v), x, (const T*)nullptr); put(v, x, same); }
    if (threadIdx.x < 2) {                          // the partial vectors
        const int pv = threadIdx.x == 0 ? 0 : g.count - 1;
        if (pv >= v0 && pv < v1 && !g.whole(pv) && (threadIdx.x == 0 || g.count > 1)) { float x[N]; g.load_part(pv, x, 0.0f); put(pv, x, false); }
    }
}

// Zeros over the vectors [v0, v1) of a row.
template <typename T>
__device__ __forceinline__ void write_zeros(T* row, int n, int v0, int v1) {
    const RowGrid<T> o(row, n);
    for (int v = v0 + threadIdx.x; v < v1 && v < o.count; v += NT) {
        if (o.whole(v)) *reinterpret_cast<uint4*>(row + o.first(v)) = make_uint4(0, 0, 0, 0);
        else
#pragma unroll
            for (int i = 0; i < RowGrid<T>::N; ++i) if (o.first(v) + i >= 0 && o.first(v) + i < n) Elem<T>::store(row, o.first(v) + i, 0.0f);
    }
}

// The vectors of CTA `part` of `parts` (a vector more than the row has: the gradient can start at another offset from a boundary).
__device__ __forceinline__ void part_of(int count, int part, int parts, int& v0, int& v1) {
    const int per = (count + parts - 1) / parts;
    v0 = min(part * per, count);
    v1 = min(v0 + per, count);
}

// A row whose weight is zero: zeros in this CTA's part.
template <typename T>
__device__ __forceinline__ void zero_part(const Args& a, int64_t row, int part, int parts) {
    T* out = reinterpret_cast<T*>(a.grad) + row * a.grad_pitch;
    const RowGrid<T> o(out, a.vocab);
    int v0, v1;
    part_of(o.count, part, parts, v0, v1);
    write_zeros(out, a.vocab, v0, v1);
}

template <typename T, int MODE>
__global__ void __launch_bounds__(NT, 2) distill_kernel(Args a) {
    constexpr int N = RowGrid<T>::N;
    extern __shared__ __align__(16) unsigned char dyn[];
    __shared__ Shared sh;
    const int C = a.cluster, rank = C > 1 ? (int)(blockIdx.x % C) : 0, t = threadIdx.x;
    const int64_t row = blockIdx.x / C;
    const float w = a.weights ? a.weights[row] : 1.0f;
    if (w == 0.0f) {                                // the row's logits are not looked at
        if (rank == 0 && t == 0) a.loss[row] = 0.0f;
        if (MODE == STEP) zero_part<T>(a, row, rank, C);
        return;
    }
    const RowGrid<T> g(reinterpret_cast<const T*>(a.logits) + row * a.pitch, a.vocab);
    int v0, v1;
    part_of(g.count, rank, C, v0, v1);
    const int e0 = max(g.first(v0), 0), e1 = min(g.first(v1), a.vocab), base = g.first(v0);     // elements of this CTA; bit 0 of the bitmap
    double* s_e = reinterpret_cast<double*>(dyn);                      // [k] exp(t_j - M), then p_j
    int* s_idx = reinterpret_cast<int*>(s_e + a.k);                    // [k]
    uint32_t* bitmap = reinterpret_cast<uint32_t*>(s_idx + (a.k + 1) / 2 * 2);
    const int words = ((v1 - v0) * N + 31) / 32;
    for (int i = t; i < words; i += NT) bitmap[i] = 0;
    if (t == 0) sh.dup = 0;

    // the list
    int idx[PER_THREAD];
    double tj[PER_THREAD], yj[PER_THREAD];
    float mt = -INF_F, mk = -INF_F;                 // largest t, largest y of this CTA's entries: as floats, only references
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        const int j = t + i * NT;
        idx[i] = -1;
        tj[i] = yj[i] = 0.0;
        if (j < a.k) {
            idx[i] = a.indices[row * a.k + j];
            if (idx[i] < 0 || idx[i] >= a.vocab) idx[i] = -1;
            s_idx[j] = idx[i];
            if (idx[i] >= 0) {
                tj[i] = list_value(a, row * a.k + j) / a.tau;
                mt = fmaxf(mt, (float)tj[i]);
                if (idx[i] >= e0 && idx[i] < e1) {
                    yj[i] = (double)Elem<T>::load(g.p, idx[i]) / a.tau;
                    mk = fmaxf(mk, (float)yj[i]);
                }
            }
        }
    }
    const double rest = a.rest ? (double)a.rest[row] : -(double)INF_F;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
        mk = fmaxf(mk, __shfl_xor_sync(0xffffffffu, mk, o));
    }
    if (lane_id() == 0) { sh.fmax[warp_id()][0] = mt; sh.fmax[warp_id()][1] = mk; }
    __syncthreads();                                // (the bitmap is clear, too)
    mt = mk = -INF_F;
    for (int i = 0; i < WARPS; ++i) { mt = fmaxf(mt, sh.fmax[i][0]); mk = fmaxf(mk, sh.fmax[i][1]); }
    mt = fmaxf(mt, (float)rest);
    const double M = mt == -INF_F ? 0.0 : (double)mt, Mk = mk == -INF_F ? 0.0 : (double)mk;
    double sum_p = 0.0, sum_k = 0.0, cross = 0.0;
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        const int j = t + i * NT;
        if (j >= a.k) continue;
        const double e = idx[i] >= 0 ? exp(tj[i] - M) : 0.0;
        s_e[j] = e;
        sum_p += e;
        if (idx[i] >= e0 && idx[i] < e1) {
            const int bit = idx[i] - base;
            const uint32_t was = atomicOr(&bitmap[bit >> 5], 1u << (bit & 31));
            if (was >> (bit & 31) & 1u) sh.dup = 1;
            else sum_k += exp(yj[i] - Mk);
            if (!(e == 0.0)) cross += e * (tj[i] - yj[i]);
        }
    }
    block_sum(sh, sum_p, sum_k, cross);             // (its barrier: the bitmap is complete)
    const double e_rest = rest == -(double)INF_F ? 0.0 : exp(rest - M);
    const double Sp = sum_p + e_rest;

    // everything else: running maximum and sum a thread
    float m = -INF_F, mr = 0.0f, s = 0.0f;
    const float scale = a.scale;
    auto add = [&](float (&x)[N], uint32_t marked) {
        if (marked) {
#pragma unroll
            for (int i = 0; i < N; ++i) if (marked >> i & 1u) x[i] = -INF_F;
        }
        float vm = x[0];
#pragma unroll
        for (int i = 1; i < N; ++i) vm = fmaxf(vm, x[i]);
        if (vm > m) {
            s *= ex2((m - vm) * scale);
            m = mr = vm;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) s += ex2((x[i] - mr) * scale);
    };
    auto marks = [&](int v) -> uint32_t {
        const int bit = (v - v0) * N;
        return reinterpret_cast<const unsigned char*>(bitmap)[bit >> 3] >> (bit & 7) & ((1u << N) - 1u);
    };
    {
        const int w0 = g.whole_from(v0), w1 = g.whole_to(v1);
        int v = w0 + t;
        for (; v + (UNROLL - 1) * NT < w1; v += UNROLL * NT) {
            uint4 r[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) r[u] = g.load(v + u * NT);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) { float x[N]; unpack(r[u], x, (const T*)nullptr); add(x, marks(v + u * NT)); }
        }
        for (; v < w1; v += NT) { float x[N]; unpack(g.load(v), x, (const T*)nullptr); add(x, marks(v)); }
        if (t < 2) {
            const int pv = t == 0 ? 0 : g.count - 1;
            if (pv >= v0 && pv < v1 && !g.whole(pv) && (t == 0 || g.count > 1)) { float x[N]; g.load_part(pv, x, -INF_F); add(x, marks(pv)); }
        }
    }
    // the block's reference and sum
    float ref = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, o));
    if (lane_id() == 0) sh.fmax[warp_id()][0] = ref;
    __syncthreads();
    ref = -INF_F;
    for (int i = 0; i < WARPS; ++i) ref = fmaxf(ref, sh.fmax[i][0]);
    if (ref == -INF_F) ref = 0.0f;
    if (!(s == 0.0f)) s *= ex2((mr - ref) * scale);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane_id() == 0) sh.fsum[warp_id()] = s;
    __syncthreads();
    if (t == 0) {
        double St = 0.0;
        for (int i = 0; i < WARPS; ++i) St += (double)sh.fsum[i];
        sh.part[0] = ref; sh.part[1] = St; sh.part[2] = Mk; sh.part[3] = sum_k; sh.part[4] = cross;
    }
    if (C > 1) cluster_arrive_wait();
    if (t == 0) {                                   // every CTA of the cluster computes the same row's numbers in the same order
        double R = -(double)INF_F, K = -(double)INF_F, St = 0.0, Sk = 0.0, B = 0.0;
        double part[5];
        auto fetch = [&](int c) { for (int i = 0; i < 5; ++i) part[i] = C > 1 ? cluster_load_f64(&sh.part[i], c) : sh.part[i]; };
        for (int c = 0; c < C; ++c) {
            fetch(c);
            if (!(part[1] == 0.0)) R = fmax(R, part[0]);
            if (!(part[3] == 0.0)) K = fmax(K, part[2]);
        }
        if (R == -(double)INF_F) R = 0.0;
        if (K == -(double)INF_F) K = 0.0;
        for (int c = 0; c < C; ++c) {
            fetch(c);
            if (!(part[1] == 0.0)) St += part[1] * exp((part[0] - R) / a.tau);
            if (!(part[3] == 0.0)) Sk += part[3] * exp(part[2] - K);
            B += part[4];
        }
        const double none = -(double)INF_F;
        const double Lt = St == 0.0 ? none : R / a.tau + log(St), Lk = Sk == 0.0 ? none : K + log(Sk);
        const double top = fmax(Lt, Lk);
        const double L = top == none ? none : top + log(exp(Lt - top) + exp(Lk - top));
        const double Lp = Sp == 0.0 ? 0.0 : M + log(Sp), inv = Sp == 0.0 ? 0.0 : 1.0 / Sp;
        const double pt = e_rest * inv, mass = sum_p * inv, P = Sp == 0.0 ? 0.0 : 1.0;
        double l = 0.0, off = 0.0;
        if (!(Sp == 0.0)) l = B * inv - Lp * mass + L * P;
        if (!(pt == 0.0)) l += St == 0.0 ? (double)INF_F : pt * (rest - Lp - Lt);
        if (!(St == 0.0)) off = (P * exp(Lt - L) - pt) / St;
        if (rank == 0) a.loss[row] = (float)(l * (double)w);
        if (rank == 0 && MODE == LOSS) a.stats[row] = make_float2((float)R, (float)off);
        sh.stat[0] = inv; sh.stat[1] = L; sh.stat[2] = P;
        sh.ref = (float)R; sh.off = (float)off;
    }
    if (C > 1) cluster_arrive_wait();               // (the other CTAs' parts stay until everybody has read them)
    else __syncthreads();

    // tau dloss/dz at this CTA's entries; an index that occurs again has the same number at every place
    const double inv = sh.stat[0], L = sh.stat[1], P = sh.stat[2];
    const float back = (float)((double)w / a.tau);
    float d[PER_THREAD];
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        const int j = t + i * NT;
        d[i] = 0.0f;
        if (j < a.k && idx[i] >= e0 && idx[i] < e1) {
            double p = s_e[j];
            if (sh.dup) {
                p = 0.0;
                for (int n = 0; n < a.k; ++n) if (s_idx[n] == idx[i]) p += s_e[n];
            }
            d[i] = (float)(P * exp(yj[i] - L) - p * inv);
            if (MODE == LOSS) a.list_grad[row * a.k + j] = d[i];
        }
    }
    if (MODE == STEP) {
        T* out = reinterpret_cast<T*>(a.grad) + row * a.grad_pitch;
        write_outside(g, v0, v1, out, sh.ref, scale, sh.off * back);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER_THREAD; ++i)
            if (t + i * NT < a.k && idx[i] >= e0 && idx[i] < e1) Elem<T>::store(out, idx[i], d[i] * back);
    }
}

// The gradient from what the loss left: one pass, several CTAs a row.
template <typename T>
__global__ void __launch_bounds__(NT, 3) distill_grad_kernel(Args a) {
    const int parts = a.cluster, part = blockIdx.x % parts, t = threadIdx.x;
    const int64_t row = blockIdx.x / parts;
    const float w = a.weights ? a.weights[row] : 1.0f;
    if (w == 0.0f) { zero_part<T>(a, row, part, parts); return; }
    const float2 st = a.stats[row];
    const float back = (float)((double)w * (double)a.grad_loss[row * a.grad_loss_stride] / a.tau);
    const RowGrid<T> g(reinterpret_cast<const T*>(a.logits) + row * a.pitch, a.vocab);
    int v0, v1;
    part_of(g.count, part, parts, v0, v1);
    const int e0 = max(g.first(v0), 0), e1 = min(g.first(v1), a.vocab);
    T* out = reinterpret_cast<T*>(a.grad) + row * a.grad_pitch;
    write_outside(g, v0, v1, out, st.x, a.scale, st.y * back);
    __syncthreads();
    for (int j = t; j < a.k; j += NT) {
        const int i = a.indices[row * a.k + j];
        if (i >= e0 && i < e1) Elem<T>::store(out, i, a.list_grad[row * a.k + j] * back);
    }
}

// CTAs of a row: as many as give every SM one, up to eight, but no part below 4 KB; and as many as its bitmap needs.
static int cluster_of(int64_t rows, int64_t bytes, int sms) {
    int c = 1;
    while (c < 8 && rows * c * 2 <= sms * 2 && bytes / (2 * c) >= 4096) c *= 2;
    return c;
}

template <typename T, int MODE> int launch(Args a, int64_t rows, cudaStream_t s) {
    const int sms = device_sm_count();
    if (sms < 0) return MAB_ERR_CUDA;
    a.cluster = cluster_of(rows, (int64_t)a.vocab * sizeof(T), sms);
    const size_t bits = ((size_t)(a.vocab + RowGrid<T>::N) / a.cluster + 2 * RowGrid<T>::N + 63) / 32 * 4;
    const size_t smem = (size_t)a.k * 8 + (size_t)(a.k + 1) / 2 * 8 + bits;
    return launch_rows(distill_kernel<T, MODE>, "distill", rows * a.cluster, NT, smem, a.cluster, s, a);
}

template <typename T> int launch_grad(Args a, int64_t rows, cudaStream_t s) {
    const int sms = device_sm_count();
    if (sms < 0) return MAB_ERR_CUDA;
    a.cluster = cluster_of(rows, (int64_t)a.vocab * sizeof(T), sms);
    return launch_rows(distill_grad_kernel<T>, "distill_grad", rows * a.cluster, NT, 0, 1, s, a);
}

static int check(const char* who, int64_t rows, int64_t vocab, int64_t k, const void* logits, int dtype, int64_t pitch, const int32_t* indices,
                 const void* values, int v_dtype, const float* rest, const float* weights, double tau) {
    MAB_REQUIRE(rows >= 0 && vocab >= 1 && k >= 1, MAB_ERR_BAD_ARG, "%s: rows=%lld, vocab=%lld, k=%lld", who, (long long)rows, (long long)vocab, (long long)k);
    MAB_REQUIRE(dtype == MAB_F32 || dtype == MAB_BF16, MAB_ERR_UNSUPPORTED, "%s: element type %d", who, dtype);
    MAB_REQUIRE(v_dtype == MAB_F32 || v_dtype == MAB_BF16, MAB_ERR_UNSUPPORTED, "%s: element type of the values %d", who, v_dtype);
    MAB_REQUIRE(tau > 1e-6 && tau < 1e6, MAB_ERR_BAD_ARG, "%s: temperature=%g outside (1e-6, 1e6)", who, tau);
    MAB_REQUIRE(rows < (1 << 28) && vocab <= MAB_MAX_VOCAB && k <= MAB_MAX_LIST, MAB_ERR_LIMIT, "%s: rows=%lld, vocab=%lld, k=%lld beyond 2^28, %d, %d",
                who, (long long)rows, (long long)vocab, (long long)k, MAB_MAX_VOCAB, MAB_MAX_LIST);
    if (rows == 0) return MAB_OK;
    MAB_REQUIRE(logits && indices && values, MAB_ERR_BAD_ARG, "%s: null pointer", who);
    MAB_REQUIRE(pitch >= vocab, MAB_ERR_BAD_ARG, "%s: rows of %lld logits lie %lld apart", who, (long long)vocab, (long long)pitch);
    MAB_REQUIRE(aligned_to(logits, dtype == MAB_F32 ? 4 : 2) && aligned_to(indices, 4) && aligned_to(values, v_dtype == MAB_F32 ? 4 : 2) &&
                aligned_to(rest, 4) && aligned_to(weights, 4), MAB_ERR_BAD_ARG, "%s: misaligned buffer", who);
    return MAB_OK;
}

// A gradient in the logits' own memory has to replace them element by element; any other overlap would be read after it was written.
static int check_grad(const char* who, int64_t rows, int64_t vocab, const void* logits, int dtype, int64_t pitch, const void* grad, int64_t grad_pitch) {
    MAB_REQUIRE(grad_pitch >= vocab, MAB_ERR_BAD_ARG, "%s: rows of %lld gradients lie %lld apart", who, (long long)vocab, (long long)grad_pitch);
    MAB_REQUIRE(aligned_to(grad, dtype == MAB_F32 ? 4 : 2), MAB_ERR_BAD_ARG, "%s: misaligned buffer", who);
    if (logits == grad && pitch == grad_pitch) return MAB_OK;
    const int64_t e = dtype == MAB_F32 ? 4 : 2;
    const uintptr_t z0 = reinterpret_cast<uintptr_t>(logits), z1 = z0 + ((rows - 1) * pitch + vocab) * e;
    const uintptr_t g0 = reinterpret_cast<uintptr_t>(grad), g1 = g0 + ((rows - 1) * grad_pitch + vocab) * e;
    MAB_REQUIRE(z1 <= g0 || g1 <= z0, MAB_ERR_BAD_ARG, "%s: the gradient overlaps the logits without being them", who);
    return MAB_OK;
}

static Args args_of(int64_t vocab, int64_t k, const void* logits, int64_t pitch, const int32_t* indices, const void* values, int v_dtype,
                    const float* rest, const float* weights, double tau) {
    Args a = {};
    a.logits = logits; a.pitch = pitch; a.indices = indices; a.values = values; a.values_bf16 = v_dtype == MAB_BF16;
    a.rest = rest; a.weights = weights; a.tau = tau; a.scale = (float)(1.4426950408889634 / tau);
    a.vocab = (int)vocab; a.k = (int)k;
    return a;
}

}  // namespace distill
}  // namespace mab

using namespace mab;

extern "C" int mab_distill_loss(int64_t rows, int64_t vocab, int64_t k, const void* logits, int dtype, int64_t pitch, const int32_t* indices,
                                const void* values, int v_dtype, const float* rest, const float* weights, double temperature, float* loss,
                                float* stats, float* list_grad, void* stream) {
    if (int rc = distill::check("mab_distill_loss", rows, vocab, k, logits, dtype, pitch, indices, values, v_dtype, rest, weights, temperature)) return rc;
    if (rows == 0) return MAB_OK;
    MAB_REQUIRE(loss && stats && list_grad, MAB_ERR_BAD_ARG, "mab_distill_loss: null pointer");
    MAB_REQUIRE(aligned_to(loss, 4) && aligned_to(stats, 8) && aligned_to(list_grad, 4), MAB_ERR_BAD_ARG, "mab_distill_loss: misaligned buffer");
    distill::Args a = distill::args_of(vocab, k, logits, pitch, indices, values, v_dtype, rest, weights, temperature);
    a.loss = loss; a.stats = reinterpret_cast<float2*>(stats); a.list_grad = list_grad;
    return dtype == MAB_F32 ? distill::launch<float, distill::LOSS>(a, rows, (cudaStream_t)stream)
                            : distill::launch<uint16_t, distill::LOSS>(a, rows, (cudaStream_t)stream);
}

extern "C" int mab_distill_grad(int64_t rows, int64_t vocab, int64_t k, const void* logits, int dtype, int64_t pitch, const int32_t* indices,
                                const float* weights, double temperature, const float* stats, const float* list_grad, const float* grad_loss,
                                int64_t grad_loss_stride, void* grad, int64_t grad_pitch, void* stream) {
    if (int rc = distill::check("mab_distill_grad", rows, vocab, k, logits, dtype, pitch, indices, list_grad, MAB_F32, nullptr, weights, temperature)) return rc;
    if (rows == 0) return MAB_OK;
    MAB_REQUIRE(stats && grad_loss && grad, MAB_ERR_BAD_ARG, "mab_distill_grad: null pointer");
    MAB_REQUIRE(grad_loss_stride >= 0, MAB_ERR_BAD_ARG, "mab_distill_grad: grad_loss_stride=%lld", (long long)grad_loss_stride);
    MAB_REQUIRE(aligned_to(stats, 8) && aligned_to(grad_loss, 4), MAB_ERR_BAD_ARG, "mab_distill_grad: misaligned buffer");
    if (int rc = distill::check_grad("mab_distill_grad", rows, vocab, logits, dtype, pitch, grad, grad_pitch)) return rc;
    distill::Args a = distill::args_of(vocab, k, logits, pitch, indices, nullptr, MAB_F32, nullptr, weights, temperature);
    a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats)); a.list_grad = const_cast<float*>(list_grad);
    a.grad_loss = grad_loss; a.grad_loss_stride = grad_loss_stride; a.grad = grad; a.grad_pitch = grad_pitch;
    return dtype == MAB_F32 ? distill::launch_grad<float>(a, rows, (cudaStream_t)stream) : distill::launch_grad<uint16_t>(a, rows, (cudaStream_t)stream);
}

extern "C" int mab_distill_step(int64_t rows, int64_t vocab, int64_t k, const void* logits, int dtype, int64_t pitch, const int32_t* indices,
                                const void* values, int v_dtype, const float* rest, const float* weights, double temperature, float* loss,
                                void* grad, int64_t grad_pitch, void* stream) {
    if (int rc = distill::check("mab_distill_step", rows, vocab, k, logits, dtype, pitch, indices, values, v_dtype, rest, weights, temperature)) return rc;
    if (rows == 0) return MAB_OK;
    MAB_REQUIRE(loss && grad, MAB_ERR_BAD_ARG, "mab_distill_step: null pointer");
    MAB_REQUIRE(aligned_to(loss, 4), MAB_ERR_BAD_ARG, "mab_distill_step: misaligned buffer");
    if (int rc = distill::check_grad("mab_distill_step", rows, vocab, logits, dtype, pitch, grad, grad_pitch)) return rc;
    distill::Args a = distill::args_of(vocab, k, logits, pitch, indices, values, v_dtype, rest, weights, temperature);
    a.loss = loss; a.grad = grad; a.grad_pitch = grad_pitch;
    return dtype == MAB_F32 ? distill::launch<float, distill::STEP>(a, rows, (cudaStream_t)stream)
                            : distill::launch<uint16_t, distill::STEP>(a, rows, (cudaStream_t)stream);
}
