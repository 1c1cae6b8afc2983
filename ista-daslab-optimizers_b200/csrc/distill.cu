// Distillation from a teacher's top logits: per row a list of k (index, logit) pairs and, where the teacher gave it, the logarithm of the
// mass of everything else (`rest`), against the student's logits z.  With t_j = value_j / tau, y_v = z_v / tau,
//
//   Lp = log(sum_j exp t_j + exp rest),  p_j = exp(t_j - Lp),  p_t = exp(rest - Lp),  P = sum_j p_j + p_t  (1, or 0 where there is nothing)
//   L = log sum_v exp y_v,  L_t = log sum_{v not in the list} exp y_v,  q_v = exp(y_v - L),  q_t = exp(L_t - L)
//   loss = sum_j p_j (log p_j - log q_j) + p_t (log p_t - log q_t)
//   tau dloss/dz_v = P q_v - sum_{j: index_j = v} p_j              for v in the list
//                  = exp(y_v - L_t) (P q_t - p_t)                  elsewhere
//
// An index that occurs again has a term of its own for each of its entries: with p = sum p_j over them, sum p_j log(p_j / q) = p log(p / q) - p H(p_j / p), H the entropy of the split.
//
// A row belongs to a cluster of one to eight CTAs, each of which has its part of the row in shared memory from the beginning to the end (a bulk copy, on its way while
// the list is worked on): one pass with a running maximum and sum, and for the gradient a second one that reads no global memory.  The list's positions are
// overwritten by -inf there, so the sum over the others is their own, not a difference of two large ones.  The k terms of the list are in 64 bits: near the
// optimum the loss is what is left of a difference, and there an error of S_t only enters with the factor q_t - p_t as long as the terms that share it are exact.
// Rows too long for that are read twice, with a bitmap of the list's positions.  The CTAs exchange six numbers through distributed shared memory, in rank order:
// results do not depend on timing.
//
// Bound by HBM and by the chain of phases around the passes (list, block and cluster sums, three logarithms: some 5 us a row, which the SM's other rows cover in part).
// bf16, rows of 128256, k = 64 (us): loss of 1536 rows 75 (5.2 TB/s), its gradient 149 (6.2 TB/s), loss and gradient of 4096 rows in one call 442 (4.7 TB/s of the two passes
// over HBM that it needs; what it holds and what L2 keeps leave 1.09 of their bytes; 569 before anything was held).
#include <initializer_list>
#include <type_traits>
#include "rows.cuh"
#include "async_copy.cuh"

namespace mab {
namespace distill {

constexpr int GRAD_NT = 512, MOST_WARPS = 16;
constexpr int MAX_K = 1024;
constexpr int UNROLL = 4;                          // vectors of 16 bytes a thread has in flight
constexpr int PART = 66 * 1024;                    // bytes of a row's part with which three CTAs share an SM
constexpr int STEP_SHARED = 108 * 1024;            // ... of shared memory with which two do
constexpr int AHEAD = 64 * 1024;                  // bytes of a row asked into L2 before the list is worked on
__device__ int g_timeout;
enum Mode { LOSS, STEP };

struct Args {
    const void* logits;
    int64_t pitch;
    const int32_t* indices;
    const void* values;
    int values_bf16;
    const float* rest;
    const float* weights;
    double inv_tau;                                // 1 / tau
    float scale;                                   // log2(e) / tau
    float* loss;
    float2* stats;                                 // per row: reference, factor of the positions outside the list (LOSS)
    float* list_grad;                              // [rows, k] tau dloss/dz at the list's positions (LOSS)
    void* grad;                                    // STEP, GRAD
    int64_t grad_pitch;
    const float* grad_loss;                        // GRAD: [rows], `grad_loss_stride` apart
    int64_t grad_loss_stride;
    int vocab, k, cluster, held;
};

struct Shared {
    uint64_t bar;
    double red[MOST_WARPS][4];
    double part[6];                                // this CTA's part, read by the cluster: reference, S_t, m_k, S_k, its entries' B and e
    double inv, q_scale, P;                        // 1 / Sp, exp(Mk - L), P
    float max_t[MOST_WARPS], max_k[MOST_WARPS], ref_w[MOST_WARPS], sum_w[MOST_WARPS];
    float ref, off;
    uint32_t edge[2];                              // the list's positions in the first and the last, partial vector
    int dup;
};

__device__ __forceinline__ float list_value(const Args& a, int64_t at) {
    return a.values_bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(a.values)[at]) : reinterpret_cast<const float*>(a.values)[at];
}

// A logit over the temperature: rounded, so that the difference of two equal ones is 0 however large they are (a fused subtraction would leave the product's rounding, 1 at 10^16).
__device__ __forceinline__ double at_tau(const Args& a, float logit) { return __dmul_rn((double)logit, a.inv_tau); }

// Sums of four doubles over the first `warps` warps, in every thread.
__device__ __forceinline__ void block_sum(Shared& sh, int warps, double& x, double& y, double& z, double& u) {
    if (warp_id() < warps) {
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            x += __shfl_xor_sync(0xffffffffu, x, o);
            y += __shfl_xor_sync(0xffffffffu, y, o);
            z += __shfl_xor_sync(0xffffffffu, z, o);
            u += __shfl_xor_sync(0xffffffffu, u, o);
        }
        if (lane_id() == 0) { sh.red[warp_id()][0] = x; sh.red[warp_id()][1] = y; sh.red[warp_id()][2] = z; sh.red[warp_id()][3] = u; }
    }
    __syncthreads();
    x = y = z = u = 0.0;
    for (int w = 0; w < warps; ++w) { x += sh.red[w][0]; y += sh.red[w][1]; z += sh.red[w][2]; u += sh.red[w][3]; }
}

// factor * exp2((x - ref) scale) of a vector.
template <typename T, int N> __device__ __forceinline__ uint4 outside(uint4 r, uint64_t ref2, uint64_t scale2, uint64_t factor2) {
    uint64_t x[N / 2];
    unpack_pairs(r, x, (const T*)nullptr);
    float y[N];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        float lo, hi;
        split(mul2(add2(x[i], ref2), scale2), lo, hi);
        split(mul2(pair_of(ex2(lo), ex2(hi)), factor2), y[2 * i], y[2 * i + 1]);
    }
    return pack(y, (const T*)nullptr);
}

// Writes that over the vectors [v0, v1) of the row; `load(v)` gives the whole ones.
template <typename T, int THREADS, typename F>
__device__ __forceinline__ void write_outside(const RowGrid<T>& g, int v0, int v1, T* out, float ref, float scale, float factor, F load) {
    constexpr int N = RowGrid<T>::N;
    const bool same = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(g.p)) & 15) == 0;
    const uint64_t ref2 = pair_of(-ref, -ref), scale2 = pair_of(scale, scale), factor2 = pair_of(factor, factor);
    auto put = [&](int v, uint4 r) {
        r = outside<T, N>(r, ref2, scale2, factor2);
        if (same) { __stcs(reinterpret_cast<uint4*>(out + g.first(v)), r); return; }
        float x[N];
        unpack(r, x, (const T*)nullptr);
#pragma unroll
        for (int i = 0; i < N; ++i) Elem<T>::store(out, g.first(v) + i, x[i]);
    };
    const int w0 = g.whole_from(v0), w1 = g.whole_to(v1);
    int v = w0 + threadIdx.x;
    for (; v + (UNROLL - 1) * THREADS < w1; v += UNROLL * THREADS) {
        uint4 r[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) r[u] = load(v + u * THREADS);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) put(v + u * THREADS, r[u]);
    }
    for (; v < w1; v += THREADS) put(v, load(v));
    if (threadIdx.x < 2) {                          // the partial vectors
        const int pv = threadIdx.x == 0 ? 0 : g.count - 1;
        if (pv >= v0 && pv < v1 && !g.whole(pv) && (threadIdx.x == 0 || g.count > 1))
            for (int i = 0; i < N; ++i) {
                const int e = g.first(pv) + i;
                if (e >= 0 && e < g.n) Elem<T>::store(out, e, factor * ex2((Elem<T>::load(g.p, e) - ref) * scale));
            }
    }
}

// Zeros over the vectors [v0, v1) of a row.
template <typename T, int THREADS>
__device__ __forceinline__ void write_zeros(T* row, int n, int v0, int v1) {
    const RowGrid<T> o(row, n);
    for (int v = v0 + threadIdx.x; v < v1 && v < o.count; v += THREADS) {
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
template <typename T, int THREADS>
__device__ __forceinline__ void zero_part(const Args& a, int64_t row, int part, int parts) {
    T* out = reinterpret_cast<T*>(a.grad) + row * a.grad_pitch;
    const RowGrid<T> o(out, a.vocab);
    int v0, v1;
    part_of(o.count, part, parts, v0, v1);
    write_zeros<T, THREADS>(out, a.vocab, v0, v1);
}

// RESIDENT: the part of the row is in shared memory; otherwise only its first `a.held` whole vectors are.  PER_THREAD: entries of the list a thread has.  Threads an
// SM (us, 1024 / 1280 / 1536): loss of 1536 rows of 128256 bf16 86 / 84 / 80, step of 2048 rows of 50257 bf16 96 / 94 / 107.
template <typename T, int MODE, bool RESIDENT, int NT, int PER_THREAD>
__global__ void __launch_bounds__(NT, (PER_THREAD > 1 ? 1024 : MODE == LOSS ? 1536 : 1280) / NT) distill_kernel(Args a) {
    constexpr int N = RowGrid<T>::N, WARPS = NT / 32;
    extern __shared__ __align__(16) unsigned char dyn[];
    __shared__ Shared sh;
    const int C = a.cluster, rank = C > 1 ? (int)(blockIdx.x % C) : 0, t = threadIdx.x, k = a.k;
    const int64_t row = blockIdx.x / C;
    kernel_before_is_done();
    const float w = a.weights ? a.weights[row] : 1.0f;
    if (w == 0.0f) {                                // the row's logits are not looked at
        if (rank == 0 && t == 0) a.loss[row] = 0.0f;
        if (MODE == STEP) zero_part<T, NT>(a, row, rank, C);
        return;
    }
    const RowGrid<T> g(reinterpret_cast<const T*>(a.logits) + row * a.pitch, a.vocab);
    int v0, v1;
    part_of(g.count, rank, C, v0, v1);
    const int w0 = g.whole_from(v0), w1 = max(w0, g.whole_to(v1));
    const int e0 = max(g.first(v0), 0), e1 = min(g.first(v1), a.vocab), base = g.first(v0);     // elements of this CTA; bit 0 of the bitmap
    const int f0 = g.first(w0), f1 = g.first(w1);                      // elements of its whole vectors
    double* s_e = reinterpret_cast<double*>(dyn);                      // [k] exp(t_j - M)
    int* s_idx = reinterpret_cast<int*>(s_e + k);                      // [k]
    uint4* part = reinterpret_cast<uint4*>(dyn + ((size_t)k * 12 + 15) / 16 * 16);               // the vectors that are held
    const int held = RESIDENT ? w1 - w0 : min(a.held, w1 - w0), h1 = w0 + held;
    uint32_t* bitmap = reinterpret_cast<uint32_t*>(part + (RESIDENT ? 0 : a.held));              // of the list's positions, where not everything is held
    // the list
    int idx[PER_THREAD];
    float vj[PER_THREAD], zj[PER_THREAD];           // the teacher's logit and the student's
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        if (i * NT >= k) break;
        const bool there = t + i * NT < k;
        idx[i] = there ? a.indices[row * k + t + i * NT] : -1;
        vj[i] = there ? list_value(a, row * k + t + i * NT) : 0.0f;
    }
    const double rest = a.rest ? (double)a.rest[row] : -(double)INF_F;
    // (the loads above are on their way)
    if (t == 0) {
        mbar_init(&sh.bar, 1);
        mbar_arrive_expect_tx(&sh.bar, (uint32_t)held * 16);
        if (held > 0) bulk_g2s(part, g.p + f0, (uint32_t)held * 16, &sh.bar);
        if (!RESIDENT && w1 > h1) prefetch_bulk_l2(g.p + g.first(h1), (uint32_t)min((w1 - h1) * 16, AHEAD));   // on its way while the list is worked on
    }
    if (!RESIDENT)
        for (int i = t; i < ((v1 - v0) * N + 31) / 32; i += NT) bitmap[i] = 0;
    if (t == 0) { sh.dup = 0; sh.edge[0] = sh.edge[1] = 0; }

    // The largest of the list, and of this CTA's entries the largest of the student's: before the temperature, so that they are exact.  (t and y as floats are infinite where a logit is the
    // type's lowest and the temperature below 1, and off by more than a double's exponential covers where it is 1e16.)
    float mt = -INF_F, mk = -INF_F;
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        if (i * NT >= k) break;
        if (idx[i] < 0 || idx[i] >= a.vocab) idx[i] = -1;
        const bool own = idx[i] >= e0 && idx[i] < e1;
        zj[i] = own ? Elem<T>::load(g.p, idx[i]) : 0.0f;
        if (t + i * NT < k) s_idx[t + i * NT] = idx[i];
        if (idx[i] >= 0) mt = fmaxf(mt, vj[i]);
        if (own) mk = fmaxf(mk, zj[i]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
        mk = fmaxf(mk, __shfl_xor_sync(0xffffffffu, mk, o));
    }
    if (lane_id() == 0) { sh.max_t[warp_id()] = mt; sh.max_k[warp_id()] = mk; }
    __syncthreads();                                // (the barrier of the copy is there, or the bitmap is clear, too)
    mt = mk = -INF_F;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) { mt = fmaxf(mt, sh.max_t[i]); mk = fmaxf(mk, sh.max_k[i]); }
    double M = fmax(at_tau(a, mt), rest);
    if (M == -(double)INF_F) M = 0.0;
    const double Mk = mk == -INF_F ? 0.0 : at_tau(a, mk);
    double sum_p = 0.0, sum_k = 0.0, cross = 0.0, own_e = 0.0, ek[PER_THREAD];
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        if (i * NT >= k) break;
        const int j = t + i * NT;
        ek[i] = 0.0;
        if (j >= k) continue;
        const double from_M = at_tau(a, vj[i]) - M, e = idx[i] >= 0 ? exp(from_M) : 0.0;
        s_e[j] = e;
        sum_p += e;
        if (idx[i] >= e0 && idx[i] < e1) {
            const double from_Mk = at_tau(a, zj[i]) - Mk;
            ek[i] = exp(from_Mk);
            own_e += e;
            // (each relative to its reference: logits of 10^16, or masked by the type's lowest value on either side, would leave nothing of the other)
            if (!(e == 0.0)) cross += e * (from_M - from_Mk);
        }
    }
    const double e_rest = rest == -(double)INF_F ? 0.0 : exp(rest - M);
    bool lost = false;
    auto arrived = [&] {
        lost = !mbar_wait(&sh.bar, 0);
        if (lost) atomicExch(&g_timeout, 1);
    };
    if (RESIDENT) arrived();
    // the list's positions leave the row; who finds one gone already has an index that occurs again (or a logit of -inf, which adds nothing)
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        if (i * NT >= k) break;
        if (!(idx[i] >= e0 && idx[i] < e1)) continue;
        bool again;
        if (!RESIDENT) {
            const int bit = idx[i] - base;
            again = atomicOr(&bitmap[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1u;
        } else if (idx[i] < f0 || idx[i] >= f1) {
            const int which = idx[i] < f0 ? 0 : 1, bit = idx[i] - (which ? f1 : g.first(0));
            again = atomicOr(&sh.edge[which], 1u << bit) >> bit & 1u;
        } else if (N == 4) {
            again = atomicExch(reinterpret_cast<uint32_t*>(part) + (idx[i] - f0), 0xFF800000u) == 0xFF800000u;
        } else {
            // (half a word; another entry can have the other half.  All 16 bits are compared: a NaN with its sign set has those of -inf, too)
            const int shift = (idx[i] - f0 & 1) * 16;
            uint32_t* word = reinterpret_cast<uint32_t*>(part) + (idx[i] - f0 >> 1);
            uint32_t seen = *reinterpret_cast<volatile uint32_t*>(word), was;
            do {
                was = seen;
                seen = atomicCAS(word, was, (was & ~(0xFFFFu << shift)) | 0xFF80u << shift);
            } while (seen != was);
            again = (was >> shift & 0xFFFFu) == 0xFF80u;
        }
        if (again) sh.dup = 1;
        else sum_k += ek[i];
    }
    block_sum(sh, min(WARPS, (k + 31) / 32), sum_p, sum_k, cross, own_e);      // (its barrier: the positions are gone)
    const double Sp = sum_p + e_rest;

    // everything else: running maximum and sum a thread
    float m = -INF_F, mr = 0.0f;
    uint64_t sum2 = 0;                              // two floats
    const float scale = a.scale;
    const uint64_t scale2 = pair_of(scale, scale);
    auto raise = [&](float vm) {
        if (vm > m) {
            const float f = ex2((m - vm) * scale);
            sum2 = mul2(sum2, pair_of(f, f));
            m = mr = vm;
        }
    };
    auto add = [&](uint4 r) {
        uint64_t x[N / 2];
        unpack_pairs(r, x, (const T*)nullptr);
        const uint64_t ref2 = pair_of(-mr, -mr);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            float lo, hi;
            split(mul2(add2(x[i], ref2), scale2), lo, hi);
            sum2 = add2(sum2, pair_of(ex2(lo), ex2(hi)));
        }
    };
    auto get = [&](int v) -> uint4 { return part[v - w0]; };
    auto marked = [&](uint4 r, int v) -> uint4 {    // without the list's positions
        if (RESIDENT) return r;
        const int bit = (v - v0) * N;
        const uint32_t marks = reinterpret_cast<const unsigned char*>(bitmap)[bit >> 3] >> (bit & 7) & ((1u << N) - 1u);
        if (!marks) return r;
        float x[N];
        unpack(r, x, (const T*)nullptr);
#pragma unroll
        for (int i = 0; i < N; ++i) if (marks >> i & 1u) x[i] = -INF_F;
        return pack(x, (const T*)nullptr);
    };
    auto run = [&](int from, int to, auto load) {
        int v = from + t;
        for (; v + (UNROLL - 1) * NT < to; v += UNROLL * NT) {
            uint4 r[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) r[u] = load(v + u * NT);
            float vm = -INF_F;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) { r[u] = marked(r[u], v + u * NT); vm = fmaxf(vm, vector_max(r[u], (const T*)nullptr)); }
            raise(vm);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) add(r[u]);
        }
        for (; v < to; v += NT) {
            const uint4 r = marked(load(v), v);
            raise(vector_max(r, (const T*)nullptr));
            add(r);
        }
    };
    {
        if (!RESIDENT) {
            // (a step reads them again, from L2 if it can: they are not a stream)
            run(h1, w1, [&](int v) { return MODE == LOSS ? g.stream(v) : g.load(v); });
            arrived();
        }
        if (RESIDENT || held > 0) run(w0, h1, get);
        if (t < 2) {                                // the partial vectors
            const int pv = t == 0 ? 0 : g.count - 1;
            if (pv >= v0 && pv < v1 && !g.whole(pv) && (t == 0 || g.count > 1))
                for (int i = 0; i < N; ++i) {
                    const int e = g.first(pv) + i;
                    if (e < 0 || e >= g.n) continue;
                    const bool gone = RESIDENT ? sh.edge[e < f0 ? 0 : 1] >> (e - (e < f0 ? g.first(0) : f1)) & 1u : bitmap[(e - base) >> 5] >> ((e - base) & 31) & 1u;
                    if (gone) continue;
                    const float x = Elem<T>::load(g.p, e);
                    raise(x);
                    sum2 = add2(sum2, pair_of(ex2((x - mr) * scale), 0.0f));
                }
        }
    }
    // the warps' references and sums, then the block's
    float s, s_hi;
    split(sum2, s, s_hi);
    s += s_hi;
    float ref = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, o));
    if (ref == -INF_F) ref = 0.0f;
    if (!(s == 0.0f)) s *= ex2((mr - ref) * scale);
    if (lost) s = __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane_id() == 0) { sh.ref_w[warp_id()] = ref; sh.sum_w[warp_id()] = s; }
    __syncthreads();
    const double none = -(double)INF_F;
    // from here the first warp: lane by lane the warps, then the CTAs of the cluster, every CTA the same in the same order
    float R = -INF_F;                               // reference of the rest, a logit
    double St = 0.0, K = none, Sk = sum_k, B = cross;
    if (warp_id() == 0) {
        const int l = lane_id();
        const float ws = l < WARPS ? sh.sum_w[l] : 0.0f, wr = ws == 0.0f ? -INF_F : sh.ref_w[l & (WARPS - 1)];
        R = wr;
#pragma unroll
        for (int o = WARPS / 2; o; o >>= 1) R = fmaxf(R, __shfl_xor_sync(0xffffffffu, R, o));
        St = ws == 0.0f ? 0.0 : (double)(ws * ex2((wr - R) * scale));
#pragma unroll
        for (int o = WARPS / 2; o; o >>= 1) St += __shfl_xor_sync(0xffffffffu, St, o);
        if (C > 1 && l == 0) { sh.part[0] = (double)R; sh.part[1] = St; sh.part[2] = Mk; sh.part[3] = sum_k; sh.part[4] = cross; sh.part[5] = own_e; }
    }
    if (C > 1) cluster_arrive_wait();
    if (warp_id() == 0) {
        const int l = lane_id();
        if (C > 1) {
            const bool there = l < C;
            const float r = there ? (float)cluster_load_f64(&sh.part[0], l) : -INF_F;
            const double st = there ? cluster_load_f64(&sh.part[1], l) : 0.0, mkk = there ? cluster_load_f64(&sh.part[2], l) : none;
            const double sk = there ? cluster_load_f64(&sh.part[3], l) : 0.0;
            const double oe = there ? cluster_load_f64(&sh.part[5], l) : 0.0;
            B = there ? cluster_load_f64(&sh.part[4], l) : 0.0;
            R = st == 0.0 ? -INF_F : r;
            K = sk == 0.0 ? none : mkk;
#pragma unroll
            for (int o = 4; o; o >>= 1) {
                R = fmaxf(R, __shfl_xor_sync(0xffffffffu, R, o));
                K = fmax(K, __shfl_xor_sync(0xffffffffu, K, o));
            }
            St = st == 0.0 ? 0.0 : st * (double)ex2((r - R) * scale);
            Sk = sk == 0.0 ? 0.0 : sk * exp(mkk - K);
#pragma unroll
            for (int o = 4; o; o >>= 1) {
                St += __shfl_xor_sync(0xffffffffu, St, o);
                Sk += __shfl_xor_sync(0xffffffffu, Sk, o);
            }
            // B relative to the one reference of all
            if (!(oe == 0.0)) B -= oe * (mkk - (Sk == 0.0 ? at_tau(a, R) : K));
#pragma unroll
            for (int o = 4; o; o >>= 1) B += __shfl_xor_sync(0xffffffffu, B, o);
        } else {
            K = sum_k == 0.0 ? none : Mk;
        }
        const bool no_rest = St == 0.0, no_list = Sk == 0.0;
        // Everything relative to A.  The factor that brings S_t there is one of fp32 (where it cannot leave its range): L and L_t share it, so its error
        // enters the loss like S_t's own.
        const double y = at_tau(a, R), A = no_list ? y : K;
        const double far = (y - A) * 1.4426950408889634;
        double Sr = St;                             // S_t relative to A
        if (!no_rest && !no_list) Sr = fabs(far) < 120.0 ? St * (double)ex2((float)far) : St * exp(fmin(y - A, 700.0));
        const double Sa = Sr + Sk;
        const bool apart = !no_rest && !no_list && !(fabs(far) < 120.0);       // S_t's logarithm is taken of itself then
        // three logarithms in three lanes
        const double lg = log(l == 0 ? Sa : l == 1 ? (apart ? St : Sr) : Sp);
        const double log_a = __shfl_sync(0xffffffffu, lg, 0), log_t = __shfl_sync(0xffffffffu, lg, 1), log_p = __shfl_sync(0xffffffffu, lg, 2);
        const bool above = apart && y - A > 700.0 && Sk == Sk;                 // the list is nothing against the rest
        const double Lt = (apart ? y - A : 0.0) + log_t, L = above ? Lt : log_a;           // relative to A, too
        const double inv = Sp == 0.0 ? 0.0 : 1.0 / Sp;
        const double pt = e_rest * inv, mass = sum_p * inv, P = Sp == 0.0 ? 0.0 : 1.0;
        double l_ = 0.0, off = 0.0;
        if (!(Sp == 0.0)) l_ = B * inv + mass * (L - log_p);
        if (!(pt == 0.0)) l_ += no_rest ? (double)INF_F : pt * ((rest - M) - log_p + (L - Lt));
        if (!no_rest) off = (P * (above ? 1.0 : Sr / Sa) - pt) / St;
        else if (no_list || !(Sk == Sk)) l_ = off = __longlong_as_double(0x7FF8000000000000ll);     // no distribution at all
        if (P == 0.0) l_ = off = 0.0;               // nothing to compare with
        if (l == 0) {
            if (rank == 0) a.loss[row] = (float)(l_ * (double)w);
            if (rank == 0 && MODE == LOSS) a.stats[row] = make_float2(P == 0.0 ? INF_F : no_rest ? 0.0f : R, (float)off);
            // q_j = exp(y_j - Mk) exp(Mk - L); where A is this CTA's own reference, the second factor is 1 / Sa
            sh.inv = inv; sh.P = P;
            sh.q_scale = !(off == off) ? off : sum_k == 0.0 ? 0.0 : Mk == A && !above ? 1.0 / Sa : exp((Mk - A) - L);
            sh.ref = no_rest ? 0.0f : R;
            sh.off = (float)off;
        }
    }
    if (C > 1) cluster_arrive_wait();               // (the other CTAs' parts stay until everybody has read them)
    else __syncthreads();

    // tau dloss/dz at this CTA's entries; an index that occurs again has the same number at every place
    const double inv = sh.inv, q_scale = sh.q_scale, P = sh.P;
    const float back = (float)((double)w * a.inv_tau);
    float d[PER_THREAD];
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        if (i * NT >= k) break;
        const int j = t + i * NT;
        d[i] = 0.0f;
        if (idx[i] >= e0 && idx[i] < e1) {
            double p = s_e[j];
            if (sh.dup) {
                p = 0.0;
                for (int n = 0; n < k; ++n) if (s_idx[n] == idx[i]) p += s_e[n];
            }
            d[i] = P == 0.0 ? 0.0f : (float)(P * (ek[i] * q_scale) - p * inv);
            if (MODE == LOSS) a.list_grad[row * k + j] = d[i];
        }
    }
    if (MODE == STEP) {
        if (P == 0.0) { zero_part<T, NT>(a, row, rank, C); return; }
        T* out = reinterpret_cast<T*>(a.grad) + row * a.grad_pitch;
        // (the last time that the row is read, and what is written is not read here: neither has to stay in L2, where the rows of the other CTAs wait)
        if (RESIDENT) {
            write_outside<T, NT>(g, v0, v1, out, sh.ref, scale, sh.off * back, get);
        } else {
            write_outside<T, NT>(g, v0, v1, out, sh.ref, scale, sh.off * back, [&](int v) {
                return v < h1 ? part[v - w0] : __ldcs(reinterpret_cast<const uint4*>(g.p + g.first(v)));
            });
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER_THREAD; ++i) {
            if (i * NT >= k) break;
            if (idx[i] >= e0 && idx[i] < e1) Elem<T>::store(out, idx[i], d[i] * back);
        }
    }
}

// The gradient from what the loss left: one pass, several CTAs a row.
template <typename T>
__global__ void __launch_bounds__(GRAD_NT, 3) distill_grad_kernel(Args a) {
    const int parts = a.cluster, part = blockIdx.x % parts, t = threadIdx.x;
    const int64_t row = blockIdx.x / parts;
    kernel_before_is_done();
    const float w = a.weights ? a.weights[row] : 1.0f;
    if (w == 0.0f) { zero_part<T, GRAD_NT>(a, row, part, parts); return; }
    const float2 st = a.stats[row];
    if (st.x == INF_F && st.y == 0.0f) { zero_part<T, GRAD_NT>(a, row, part, parts); return; }      // a row without a teacher
    const float back = (float)((double)w * (double)a.grad_loss[row * a.grad_loss_stride] * a.inv_tau);
    const RowGrid<T> g(reinterpret_cast<const T*>(a.logits) + row * a.pitch, a.vocab);
    int v0, v1;
    part_of(g.count, part, parts, v0, v1);
    const int e0 = max(g.first(v0), 0), e1 = min(g.first(v1), a.vocab);
    T* out = reinterpret_cast<T*>(a.grad) + row * a.grad_pitch;
    write_outside<T, GRAD_NT>(g, v0, v1, out, st.x, a.scale, st.y * back, [&](int v) { return g.load(v); });
    __syncthreads();
    for (int j = t; j < a.k; j += GRAD_NT) {
        const int i = a.indices[row * a.k + j];
        if (i >= e0 && i < e1) Elem<T>::store(out, i, a.list_grad[row * a.k + j] * back);
    }
}

// CTAs of a row: as many as give every SM two or three, up to eight, but no part below 4 KB.
static int cluster_of(int64_t rows, int64_t bytes, int sms) {
    int c = 1;
    while (c < 8 && rows * c * 2 <= sms * 3 && bytes / (2 * c) >= 4096) c *= 2;
    return c;
}

// Parts of up to 66 KB are held as a whole, by clusters of four where a step has few rows (us, one CTA a row and four: 300 rows of 128256 bf16 52 and 47, 600 rows 83
// and 85: a cluster's exchange costs some 2 us a row; the border of 296 rows lies below both, what is best between them goes by how the waves fall and is not measured).  Longer rows: the loss reads its row once anyway; a step reads what it does not hold a second time, from L2 if the
// rows under way fit there.  Up to 140 KB they do with four CTAs of 256 threads an SM (2048 rows of 50257 bf16: 93 to 97, with two of 512 threads that hold 100 KB each 114; of
// 80000: 153 and 147), beyond 400 KB a part only with more CTAs a row (1000 rows of 151936 fp32: 325, with two 266, with four 262).
template <typename T, int MODE> int launch(Args a, int64_t rows, cudaStream_t s) {
    const int sms = device_sm_count();
    if (sms < 0) return MAB_ERR_CUDA;
    constexpr int N = RowGrid<T>::N;
    const int64_t bytes = (int64_t)a.vocab * sizeof(T);
    a.cluster = cluster_of(rows, bytes, sms);
    if (MODE == STEP) {
        int whole = a.cluster;                      // CTAs that hold the row
        while (whole < 4 && bytes / whole > PART - 64) whole *= 2;
        if (bytes / whole <= PART - 64 && rows * whole <= sms * 8) a.cluster = whole;
        while (a.cluster < 8 && bytes / a.cluster > 400 * 1024) a.cluster *= 2;
    }
    const size_t list = ((size_t)a.k * 12 + 15) / 16 * 16;
    const size_t vectors = ((size_t)a.vocab / N + 2 + a.cluster - 1) / a.cluster, bits = (vectors * N + 31) / 32 * 4;
    auto go = [&](auto resident, auto threads, size_t smem) {
        constexpr bool RESIDENT = decltype(resident)::value;
        constexpr int NT = decltype(threads)::value;
        // (lists of up to an entry a thread leave registers for another CTA)
        auto* kernel = a.k <= NT ? distill_kernel<T, MODE, RESIDENT, NT, 1> : distill_kernel<T, MODE, RESIDENT, NT, MAX_K / NT>;
        return launch_rows(kernel, "distill", rows * a.cluster, NT, list + smem, a.cluster, s, a);
    };
    if (vectors * 16 <= PART) return go(std::true_type(), std::integral_constant<int, 256>(), vectors * 16);
    if constexpr (MODE == STEP)
        if (vectors * 16 > 140 * 1024) {
            a.held = (int)std::min<int64_t>((int64_t)vectors, std::max<int64_t>(0, STEP_SHARED - (int64_t)(list + bits)) / 16);
            return go(std::false_type(), std::integral_constant<int, 512>(), bits + (size_t)a.held * 16);
        }
    return go(std::false_type(), std::integral_constant<int, 256>(), bits);
}

template <typename T> int launch_grad(Args a, int64_t rows, cudaStream_t s) {
    const int sms = device_sm_count();
    if (sms < 0) return MAB_ERR_CUDA;
    a.cluster = cluster_of(rows, (int64_t)a.vocab * sizeof(T), sms);
    return launch_rows(distill_grad_kernel<T>, "distill_grad", rows * a.cluster, GRAD_NT, 0, 1, s, a);
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

// ... and one that lies over the lists or the rows' numbers, too.
static int check_apart(const char* who, int64_t rows, int64_t vocab, int64_t k, int dtype, const void* grad, int64_t grad_pitch, const int32_t* indices,
                       std::initializer_list<Span> others) {
    const int64_t e = dtype == MAB_F32 ? 4 : 2;
    const Span g = {grad, rows, vocab * e, grad_pitch * e};
    bool ok = apart(g, vector_span(indices, rows * k * 4));
    for (const Span& o : others) ok = ok && apart(g, o);
    MAB_REQUIRE(ok, MAB_ERR_BAD_ARG, "%s: the gradient overlaps the lists or the rows' numbers", who);
    return MAB_OK;
}

static Args args_of(int64_t vocab, int64_t k, const void* logits, int64_t pitch, const int32_t* indices, const void* values, int v_dtype,
                    const float* rest, const float* weights, double tau) {
    Args a = {};
    a.logits = logits; a.pitch = pitch; a.indices = indices; a.values = values; a.values_bf16 = v_dtype == MAB_BF16;
    a.rest = rest; a.weights = weights; a.inv_tau = 1.0 / tau; a.scale = (float)(1.4426950408889634 / tau);
    a.vocab = (int)vocab; a.k = (int)k;
    return a;
}

}  // namespace distill

int copy_timeout_distill(int* out, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(out, distill::g_timeout, sizeof(int));
    if (e == cudaSuccess && clear) { const int z = 0; e = cudaMemcpyToSymbol(distill::g_timeout, &z, sizeof(int)); }
    return e == cudaSuccess ? MAB_OK : cuda_fail(e, "distill wait flag");
}

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
    if (int rc = distill::check_apart("mab_distill_grad", rows, vocab, k, dtype, grad, grad_pitch, indices,
                                      {vector_span(list_grad, rows * k * 4), vector_span(stats, rows * 8), vector_span(weights, rows * 4),
                                       vector_span(grad_loss, ((rows - 1) * grad_loss_stride + 1) * 4)})) return rc;
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
    if (int rc = distill::check_apart("mab_distill_step", rows, vocab, k, dtype, grad, grad_pitch, indices,
                                      {vector_span(values, rows * k * (v_dtype == MAB_F32 ? 4 : 2)), vector_span(rest, rows * 4), vector_span(weights, rows * 4),
                                       vector_span(loss, rows * 4)})) return rc;
    distill::Args a = distill::args_of(vocab, k, logits, pitch, indices, values, v_dtype, rest, weights, temperature);
    a.loss = loss; a.grad = grad; a.grad_pitch = grad_pitch;
    return dtype == MAB_F32 ? distill::launch<float, distill::STEP>(a, rows, (cudaStream_t)stream)
                            : distill::launch<uint16_t, distill::STEP>(a, rows, (cudaStream_t)stream);
}
