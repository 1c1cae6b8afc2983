// The k largest logits of every row, in descending order (ties: the lower index first), and rest = log sum exp(z / tau) over all others.
//
// One pass over the row.  A sample (the maxima of vectors spread over the row) gives a bound that at least k values reach: the k-th largest of the maxima.  Then the row
// streams by: a vector with a value above the bound is put on a list, every other one goes into the sum at once, relative to the bound, so the sum over the rest
// is its own and not a difference of two large ones.  The k-th largest of the listed vectors' maxima is a second, nearer bound; the listed values above it are the candidates
// (some k plus ties), the others join the sum, and the candidates are put in order.  No barrier and no decision of the block falls into the stream: where
// more come than there is room for (equal values, a row that is not like its sample), the row is gone through again, chunk by chunk, each selected from exactly in registers.
//
// The order is that of 64-bit keys, value above 2^32 - 1 - index: distinct, so "larger" contains the tie rule.  NaN lies below -inf and makes
// the rest NaN.  A row belongs to a cluster of one to eight CTAs; the first of them merges the candidates of all.
//
// Bound by the chains of phases around the stream (about a quarter of a row's time with six rows on an SM), by the special-function units, which an exponential
// per logit keeps busy for 75 us of 2048 x 128256 bf16, and by the sample's second reading: that takes 109 us with k = 64 (4.8 TB/s; the stream alone 84, plain reading 78), 93
// with k = 10; 5 x 50257 fp32 with k = 20 10.1.  Further from the bytes are lists above 128, whose bounds are found a bit a step and which a network sorts (4096 x 128256, k = 256: 429, 2.4 TB/s;
// 2048 x 20000, k = 130: 98), and short rows, which the sample reads whole before the stream does (2048 x 8000, k = 64: 33).
#include "rows.cuh"

namespace mab {
namespace toplogits {

constexpr int UNROLL = 6;                          // vectors a thread has in flight (2048 rows of 128256 bf16, k = 64, with 3 .. 8: 114, 111, 110, 109, 111, 116 us)
constexpr int SLOW_UNROLL = 2;                     // vectors a thread holds of a chunk that is selected from exactly
constexpr int MAX_K = 1024;

// Lists of up to 128 by CTAs of 256 threads, six on an SM: their chains of phases overlap the others' streams.  They keep the listed vectors themselves (the case above: 122 us
// when they were read again, from L2 or beyond; 121 with 31 KB a CTA, which leave too little of the SM's memory to the loads under way).
template <bool LARGE> struct Form {
    static constexpr int NT = LARGE ? 512 : 256, WARPS = NT / 32, CTAS = LARGE ? 3 : 6;
    static constexpr int CAP = LARGE ? 2560 : 768;             // candidates
    static constexpr int LIST = LARGE ? 2560 : 896;            // vectors that hold one by the first bound
    static constexpr int REACH = LARGE ? 1536 : 512;            // vectors that hold one by the second bound
    static constexpr bool KEPT = !LARGE;
    static constexpr int MOST_K = LARGE ? MAX_K : 128, ITEMS = CAP / NT;
    static_assert(2 * MOST_K <= CAP, "what is held and what a chunk adds have room");
};

struct Args {
    const void* logits;
    int64_t pitch;
    void* values;
    int32_t* indices;
    float* rest;
    double tau;
    float scale;
    int vocab, k, cluster, groups, per;
};

template <class F> struct Shared {
    unsigned long long cand[F::CAP];
    uint4 data[F::KEPT ? F::LIST : 1];              // vectors with a value above the bound (LARGE: not kept) ...
    int list[F::LIST];                              // ... which they are ...
    uint32_t list_key[F::LIST];                     // ... and the keys of their largest
    int reach[F::REACH];                               // those that reach the second bound
    int n_list, n_reach;
    double red[F::WARPS];
    double peer_sum[8], peer_ref[8];                // of the cluster's CTAs: sum over the rest, its reference (infinite: far), number of candidates
    uint32_t peer_n[8];
    int n;                                          // candidates (counts beyond F::CAP where they do not fit)
    int count[64];                                  // counters of a bisection, one per step
    uint32_t warp_max[F::WARPS], found;
    int scan[40];
    double terms[F::WARPS];                            // of candidates that go into the rest
};

// Order keys of as many bits as the type has; NaN (0) below -inf, one key for the two zeros.
template <typename T> struct Key {
    static constexpr int SHIFT = 32 - 8 * (int)sizeof(T);
    static constexpr uint32_t NEG_INF = KEY_NEG_INF >> SHIFT, MOST = 0xFFFFFFFFu >> SHIFT;
    __device__ __forceinline__ static uint32_t of(float x) { return row_key(x) >> SHIFT; }
    __device__ __forceinline__ static float value(uint32_t key) {
        return SHIFT ? ord_value(key << SHIFT | (key & 0x8000u ? 0u : 0xFFFFu)) : ord_value(key);
    }
    __device__ __forceinline__ static float below(uint32_t key) {              // the next value below; the key under that of +0 is the unused one of -0
        return value(key == (0x80000000u >> SHIFT) ? key - 2 : key - 1);
    }
    __device__ __forceinline__ static float bound(uint32_t key) { return key > NEG_INF ? value(key) : -INF_F; }
    __device__ __forceinline__ static unsigned long long composite(float x, int e) { return (unsigned long long)of(x) << 32 | (0xFFFFFFFFu - (uint32_t)e); }
    __device__ __forceinline__ static float value_of(unsigned long long c) { return value((uint32_t)(c >> 32)); }
};
__device__ __forceinline__ int index_of(unsigned long long c) { return (int)(0xFFFFFFFFu - (uint32_t)c); }

// A thread's sum over the rest, relative to exp2(ref), ref a reference times `scale`: exp2(x scale - ref) is one operation and the instruction, and the
// rounding of ref cancels in the end.  `far`: a reference so large was in use that its rounding is no longer small against 1: the sum does not count.
constexpr float FAR = 1048576.0f;
struct Rest {
    float s, ref, scale;
    bool far;
    __device__ __forceinline__ void add(float x) { s += ex2(fmaf(x, scale, -ref)); }
    // The reference only rises: a later bound may be lower than it (of merged lists the k-th to (k + slack)-th is any value in between, far below one's own bound), and
    // s times a power of two of the difference would overflow.  What is added later lies below some bound before it, and so below the reference.
    __device__ __forceinline__ void move(float to_value) {
        const float to = to_value == -INF_F ? -3e38f : fminf(fmaxf(to_value * scale, -3e38f), 3e38f);
        far |= to_value != -INF_F && !(fabsf(to) < FAR);
        if (to > ref) {
            if (!(s == 0.0f)) s *= ex2(ref - to);
            ref = to;
        }
    }
};

// A candidate's term in the rest, rounded to a multiple of 2^-38: candidates come in any order and to any thread, and doubles on one grid
// have the same sum in every order (32768 of them, each at most 1 but for a rounding, stay exact).
__device__ __forceinline__ double on_grid(float term) { return __dadd_rn(__dadd_rn((double)term, 24576.0), -24576.0); }
__device__ __forceinline__ double grid_term(const Rest& rest, float x) { return on_grid(ex2(fmaf(x, rest.scale, -rest.ref))); }
// Adds the block's terms to the rest, in the first thread.
template <class F> __device__ __forceinline__ void add_terms(double* parts, double mine, Rest& rest) {
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane_id() == 0) parts[warp_id()] = mine;
    __syncthreads();
    if (warp_id() == 0) {
        double all = lane_id() < F::WARPS ? parts[lane_id()] : 0.0;
#pragma unroll
        for (int o = F::WARPS / 2; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        if (lane_id() == 0) rest.s += (float)all;
    }
}

// Sum of one int per thread, step `i` of a bisection: counters are cleared by `clear_counts`, each is used once.
template <class F> __device__ __forceinline__ int block_count(Shared<F>& sh, int c, int i) {
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane_id() == 0 && c) atomicAdd(&sh.count[i], c);
    __syncthreads();
    return sh.count[i];
}
template <class F> __device__ __forceinline__ void clear_counts(Shared<F>& sh) {
    __syncthreads();
    if (threadIdx.x < 64) sh.count[threadIdx.x] = 0;
    __syncthreads();
}

// Largest key T in [lo, hi] with count(>= T) >= k, or any with count(>= T) in [k, most], `counted(mid)` being the calling thread's number of keys >= mid.
// Needs count(>= lo) >= k, count(> hi) < k.  `reached`: count(>= T).
template <class F, typename G> __device__ __forceinline__ uint32_t kth_key(Shared<F>& sh, uint32_t lo, uint32_t hi, int k, int most, int& reached, G counted) {
    clear_counts(sh);
    reached = 0x7FFFFFFF;
    for (int i = 0; lo < hi; ++i) {
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        const int c = block_count(sh, counted(mid), i);
        if (c < k) { hi = mid - 1; continue; }
        lo = mid;
        reached = c;
        if (c <= most) break;
    }
    return lo;
}

// The same for keys[0 .. n) in shared memory, n <= 32 PER, by the first warp alone: no barrier in its steps, and the other warps' slots are free for the SM's other
// CTAs.  The range is first narrowed in growing steps from where the answer is expected.  The answer is in every thread after the barrier at the end.
template <typename T, bool FROM_TOP, int PER, class F> __device__ __forceinline__ uint32_t kth_by_warp(Shared<F>& sh, const uint32_t* keys, int n, uint32_t lo, uint32_t hi, int k, int most) {
    if (warp_id() == 0) {
        uint32_t key[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = lane_id() + 32 * i < n ? keys[lane_id() + 32 * i] : 0u;         // (0 is below every mid)
        uint32_t step = 128u << (16 - Key<T>::SHIFT);              // an octave
        bool narrowing = true;
        while (lo < hi) {
            uint32_t mid = lo + (hi - lo) / 2 + 1;
            if (narrowing && (hi - lo) / 2 > step) mid = FROM_TOP ? hi - step : lo + step;
            else narrowing = false;
            step *= 2;
            int q[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < PER; ++i) q[i & 3] += key[i] >= mid;
            const int r = __reduce_add_sync(0xffffffffu, q[0] + q[1] + (q[2] + q[3]));
            if (r < k) { hi = mid - 1; narrowing &= FROM_TOP; continue; }
            lo = mid;
            narrowing &= !FROM_TOP;
            if (r <= most) break;
        }
        if (lane_id() == 0) sh.found = lo;
    }
    __syncthreads();
    return sh.found;
}

// The key of the k-th largest of n >= k keys, or one between that and the (k + slack)-th; all lie in [lo, hi], n <= F::LIST.
template <typename T, class F> __device__ __noinline__ uint32_t kth_of_list(Shared<F>& sh, int n, int k, int slack, uint32_t lo, uint32_t hi) {
    const int t = threadIdx.x;
    if (n <= k + slack + 16) return lo;             // (the sample was the whole part, or nearly)
    if (n <= 512) return kth_by_warp<T, false, 16>(sh, sh.list_key, n, lo, hi, k, k + slack);
    if (n <= 1024) return kth_by_warp<T, false, 32>(sh, sh.list_key, n, lo, hi, k, k + slack);
    int reached;
    return kth_key(sh, lo, hi, k, k + slack, reached, [&](uint32_t mid) {
        int r = 0;
        for (int i = t; i < n; i += F::NT) r += sh.list_key[i] >= mid;
        return r;
    });
}

// A key that at least k values of the whole vectors [w0, w1) reach, near the k-th largest: of the maxima of `groups` groups a thread of `per` vectors each, spread
// evenly over them.  NEG_INF where there are not enough.
template <typename T, class F> __device__ __noinline__ uint32_t bound_of_sample(Shared<F>& sh, const RowGrid<T>& g, int w0, int w1, int k, int groups, int per) {
    using K = Key<T>;
    const int total = groups * per, every = (max(w1 - w0, 0) + 31) / 32, runs = min(total * F::WARPS, every), apart = runs ? every / runs * 32 : 0;
    auto maximum = [&](int u) {                     // of the u-th vector of this thread
        const int j = u * F::WARPS + warp_id(), v = w0 + j * apart + lane_id();
        return u < total && j < runs && v < w1 ? vector_max(g.load(v), (const T*)nullptr) : -INF_F;
    };
    uint32_t top = 0;
    float m[4], of_group = -INF_F;
    int in_group = 0, group = 0;
    for (int b = 0; b < total; b += 4) {
#pragma unroll
        for (int u = 0; u < 4; ++u) m[u] = maximum(b + u);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (b + u >= total) break;
            of_group = fmaxf(of_group, m[u]);
            if (++in_group == per) {
                const uint32_t key = K::of(of_group);
                sh.list_key[group++ * F::NT + threadIdx.x] = key;
                top = max(top, key);
                in_group = 0;
                of_group = -INF_F;
            }
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane_id() == 0) sh.warp_max[warp_id()] = top;
    __syncthreads();
    top = max(__reduce_max_sync(0xffffffffu, sh.warp_max[lane_id() & (F::WARPS - 1)]), K::NEG_INF);
    const int n = groups * F::NT;
    if (n <= 256) return kth_by_warp<T, true, 8>(sh, sh.list_key, n, K::NEG_INF, top, k, k + k / 8);
    if (n <= 512) return kth_by_warp<T, true, 16>(sh, sh.list_key, n, K::NEG_INF, top, k, k + k / 8);
    if (n <= 1024) return kth_by_warp<T, true, 32>(sh, sh.list_key, n, K::NEG_INF, top, k, k + k / 8);
    int reached;
    return kth_key(sh, K::NEG_INF, top, k, k + k / 8, reached, [&](uint32_t mid) {
        int r = 0;
        for (int i = threadIdx.x; i < n; i += F::NT) r += sh.list_key[i] >= mid;
        return r;
    });
}

// Of the n > k candidates (n <= F::CAP) those from the k-th on stay, in no order, k to k + slack of them; the others go into the rest, relative to a bound below
// the former.  Returns the bound's key; [lo, hi] holds all keys.
template <typename T, class F> __device__ __noinline__ uint32_t prune(Shared<F>& sh, int k, int slack, uint32_t lo, uint32_t hi, Rest& rest) {
    const int t = threadIdx.x, n = sh.n;
    unsigned long long c[F::ITEMS];
    int reached;
#pragma unroll
    for (int i = 0; i < F::ITEMS; ++i) c[i] = t + i * F::NT < n ? sh.cand[t + i * F::NT] : 0ull;
    const uint32_t key = kth_key(sh, lo, hi, k, k + slack, reached, [&](uint32_t mid) {
        int r = 0;
#pragma unroll
        for (int i = 0; i < F::ITEMS; ++i) {
            if (i * F::NT >= n) break;
            r += t + i * F::NT < n && (uint32_t)(c[i] >> 32) >= mid;
        }
        return r;
    });
    unsigned long long last = (unsigned long long)key << 32;
    if (reached > k + slack) {                      // more equals of the k-th than places: the lowest indices
        clear_counts(sh);
        int above = 0;
#pragma unroll
        for (int i = 0; i < F::ITEMS; ++i) above += t + i * F::NT < n && (uint32_t)(c[i] >> 32) > key;
        above = block_count(sh, above, 0);
        last |= kth_key(sh, 0xFFFFFFFFu - (uint32_t)MAB_MAX_VOCAB, 0xFFFFFFFFu, k - above, k - above, reached, [&](uint32_t mid) {
            int r = 0;
#pragma unroll
            for (int i = 0; i < F::ITEMS; ++i) r += t + i * F::NT < n && (uint32_t)(c[i] >> 32) == key && (uint32_t)c[i] >= mid;
            return r;
        });
    }
    __syncthreads();
    if (t == 0) sh.n = 0;
    __syncthreads();
    rest.move(Key<T>::bound(key));
    double terms = 0.0;
#pragma unroll
    for (int i = 0; i < F::ITEMS; ++i) {
        if (t + i * F::NT >= n) break;
        if (c[i] >= last) sh.cand[atomicAdd(&sh.n, 1)] = c[i];
        else terms += grid_term(rest, Key<T>::value_of(c[i]));
    }
    add_terms<F>(sh.terms, terms, rest);
    return key;
}

// The candidates and the rest of the vectors [v0, v1), whatever they hold: every chunk's k largest that lie above the bound are found exactly, in
// registers; the bound is the k-th of the chunk before, and of all candidates whenever those outgrow their room.
template <typename T, class F> __device__ __noinline__ void select_slowly(Shared<F>& sh, const RowGrid<T>& g, int v0, int v1, int k, Rest& rest) {
    constexpr int N = RowGrid<T>::N;
    using K = Key<T>;
    const int t = threadIdx.x;
    __syncthreads();
    if (t == 0) sh.n = 0;
    rest.s = 0.0f;
    rest.ref = -INF_F;
    uint32_t floor_key = 0;                         // smaller keys cannot be among the k largest any more
    for (int base = v0; base < v1; base += F::NT * SLOW_UNROLL) {
        float x[SLOW_UNROLL][N];
        uint32_t valid[SLOW_UNROLL];                // bits of the elements that are there
#pragma unroll
        for (int u = 0; u < SLOW_UNROLL; ++u) {
            const int v = base + u * F::NT + t;
            valid[u] = 0;
            if (v < v1) {
                if (g.whole(v)) unpack(g.load(v), x[u], (const T*)nullptr);
                else g.load_part(v, x[u], 0.0f);
#pragma unroll
                for (int i = 0; i < N; ++i) if (g.first(v) + i >= 0 && g.first(v) + i < g.n) valid[u] |= 1u << i;
            }
        }
        auto counted = [&](uint32_t mid) {
            int r = 0;
#pragma unroll
            for (int u = 0; u < SLOW_UNROLL; ++u)
#pragma unroll
                for (int i = 0; i < N; ++i) r += (valid[u] >> i & 1u) && K::of(x[u][i]) >= mid;
            return r;
        };
        clear_counts(sh);
        const int eligible = block_count(sh, counted(floor_key), 0);
        uint32_t kth = floor_key;
        int need = 0x7FFFFFFF;                      // equals of the k-th that are taken, in the order of their indices
        if (eligible > k) {
            int reached;
            kth = kth_key(sh, floor_key, K::MOST, k, 0, reached, counted);
            clear_counts(sh);
            need = k - block_count(sh, counted(kth + 1u), 0);
            rest.move(K::bound(kth));
        }
#pragma unroll
        for (int u = 0; u < SLOW_UNROLL; ++u) {
            int equal = 0, total = 0, before = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) equal += (valid[u] >> i & 1u) && K::of(x[u][i]) == kth;
            if (need != 0x7FFFFFFF) before = block_exclusive_scan(equal, sh.scan, total);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!(valid[u] >> i & 1u)) continue;
                const uint32_t key = K::of(x[u][i]);
                if (key > kth || (key == kth && (need == 0x7FFFFFFF || before++ < need)))
                    sh.cand[atomicAdd(&sh.n, 1)] = K::composite(x[u][i], g.first(base + u * F::NT + t) + i);
                else rest.add(x[u][i]);
            }
            if (need != 0x7FFFFFFF) need = max(0, need - total);
            __syncthreads();
        }
        if (eligible > k) floor_key = kth + 1u;     // k values from the k-th on are held, with lower indices than all that follow
        if (sh.n > F::CAP - k) floor_key = prune<T>(sh, k, 0, 0u, K::MOST, rest) + 1u;
    }
    __syncthreads();
}

// Descending, n <= MAX_K with zeros behind them up to a power of two, in place.  A stage of a distance of up to 32 stays in the 64 elements that a warp has, so only
// the others need the whole block's barrier.
template <class F> __device__ __forceinline__ void sort_descending(unsigned long long* cand, int n) {
    int size = 64;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += F::NT) cand[i] = 0ull;
    int before = size;
    for (int block = 2; block <= size; block *= 2)
        for (int d = block / 2; d; d /= 2) {
            if (d > 32 || before > 32) __syncthreads();
            else __syncwarp();
            before = d;
            for (int i = threadIdx.x; i < size / 2; i += F::NT) {
                const int p = 2 * i - (i & (d - 1)), q = p + d;
                const unsigned long long x = cand[p], y = cand[q];
                if ((x < y) == ((p & block) == 0)) { cand[p] = y; cand[q] = x; }
            }
        }
    __syncthreads();
}

template <typename T, class F>
__global__ void __launch_bounds__(F::NT, F::CTAS) topk_logits_kernel(Args a) {
    constexpr int N = RowGrid<T>::N;
    using K = Key<T>;
    extern __shared__ __align__(16) unsigned char dyn[];
    Shared<F>& sh = *reinterpret_cast<Shared<F>*>(dyn);
    const int C = a.cluster, rank = C > 1 ? (int)(blockIdx.x % C) : 0, t = threadIdx.x, k = a.k;
    if (C > 1) cluster_arrive();
    const int64_t row = blockIdx.x / C;
    const RowGrid<T> g(reinterpret_cast<const T*>(a.logits) + row * a.pitch, a.vocab);
    const int per = (g.count + C - 1) / C, v0 = min(rank * per, g.count), v1 = min(v0 + per, g.count);
    const int w0 = g.whole_from(v0), w1 = g.whole_to(v1);
    if (t == 0) sh.n = sh.n_list = sh.n_reach = 0;
    kernel_before_is_done();
    Rest rest = {0.0f, -INF_F, a.scale, false};
    float bound = -INF_F;                           // values above it are candidates
    uint32_t lo_key = 0, top_key = K::MOST;         // no candidate's key lies outside
    bool slow = false;
    const bool all = (v1 - v0) * N <= F::CAP;          // everything is a candidate

    if (!all) {
        const uint32_t at = bound_of_sample<T>(sh, g, w0, w1, k, a.groups, a.per);
        slow = at == K::NEG_INF;                    // fewer than k numbers among the maxima
        if (!slow) {
            bound = K::below(at);
            lo_key = at;
            rest.move(bound);
        }
    }
    __syncthreads();
    if (!slow) {
        uint64_t sum = 0;                           // two floats
        const uint64_t scale2 = pair_of(a.scale, a.scale), ref2 = pair_of(-rest.ref, -rest.ref);
        auto see = [&](uint4 r, int v) {
            const float m = vector_max(r, (const T*)nullptr);
            if (m > bound) {
                const int at = atomicAdd(&sh.n_list, 1);
                if (at < F::LIST) {
                    sh.list[at] = v;
                    sh.list_key[at] = K::of(m);
                    if (F::KEPT) sh.data[at] = r;
                }
            } else {
                uint64_t x[N / 2];
                unpack_pairs(r, x, (const T*)nullptr);
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    float lo, hi;
                    split(fma2(x[i], scale2, ref2), lo, hi);
                    sum = add2(sum, pair_of(ex2(lo), ex2(hi)));
                }
            }
        };
        auto push = [&](float x, int e) {
            const int at = atomicAdd(&sh.n, 1);
            if (at < F::CAP) sh.cand[at] = K::composite(x, e);
        };
        if (!all) {
            int v = w0 + t;
            for (; v + (UNROLL - 1) * F::NT < w1; v += UNROLL * F::NT) {
                uint4 r[UNROLL];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) r[u] = g.stream(v + u * F::NT);
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) see(r[u], v + u * F::NT);
            }
            for (; v < w1; v += F::NT) see(g.stream(v), v);
        }
        float lo, hi;
        split(sum, lo, hi);
        rest.s += lo + hi;
        __syncthreads();
        // the vectors of the list (or all), element by element.  As many vectors as k reach the k-th of their largest: a bound nearer to the k-th value
        const int listed = all ? w1 - w0 : sh.n_list;
        slow = listed > F::LIST;
        if (!slow && !all) {
            lo_key = kth_of_list<T>(sh, listed, k, k / 8, lo_key, top_key);
            bound = K::below(lo_key);
            rest.move(bound);
        }
        double terms = 0.0;
        if (all) {
            for (int i = t; i < listed * N; i += F::NT) push(Elem<T>::load(g.p, g.first(w0) + i), g.first(w0) + i);
        } else if (!slow) {
            // vectors below the new bound go into the sum, each by its own sum in a fixed order; of the others, which are some k, a thread has an element at a time
            for (int j = t; j < listed; j += F::NT) {
                if (sh.list_key[j] >= lo_key) {
                    const int at = atomicAdd(&sh.n_reach, 1);
                    if (at < F::REACH) sh.reach[at] = j;
                    continue;
                }
                float x[N], part = 0.0f;
                unpack(F::KEPT ? sh.data[j] : g.load(sh.list[j]), x, (const T*)nullptr);
#pragma unroll
                for (int i = 0; i < N; ++i) part += ex2(fmaf(x[i], rest.scale, -rest.ref));
                terms += on_grid(part);
            }
            __syncthreads();
            const int reaching = sh.n_reach;
            slow = reaching > F::REACH;
            if (!slow)
                for (int i = t; i < reaching * N; i += F::NT) {
                    const int j = sh.reach[i / N], e = g.first(sh.list[j]) + i % N;
                    const float x = F::KEPT ? Elem<T>::load(reinterpret_cast<const T*>(&sh.data[j]), i % N) : Elem<T>::load(g.p, e);
                    if (x > bound) push(x, e);
                    else terms += grid_term(rest, x);
                }
        }
        if (t < 2) {                                // the partial vectors
            const int pv = t == 0 ? 0 : g.count - 1;
            if (pv >= v0 && pv < v1 && !g.whole(pv) && (t == 0 || g.count > 1)) {
                for (int i = 0; i < N; ++i) {
                    const int e = g.first(pv) + i;
                    if (e < 0 || e >= g.n) continue;
                    const float x = Elem<T>::load(g.p, e);
                    if (all || x > bound) push(x, e);
                    else rest.add(x);
                }
            }
        }
        add_terms<F>(sh.terms, terms, rest);
        slow |= sh.n > F::CAP;
    }
    if (slow) {
        select_slowly<T>(sh, g, v0, v1, k, rest);
        lo_key = 0;
    }

    if (C > 1) {                                    // the first CTA takes over the others' candidates and sums
        if (sh.n > F::CAP / C) prune<T>(sh, k, F::CAP / C - k, lo_key, K::MOST, rest);      // (what all of them have fits the first one's room)
        lo_key = 0;                                 // (the others' bounds are others)
        float s = rest.s;
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane_id() == 0) sh.red[warp_id()] = (double)s;
        __syncthreads();
        cluster_wait();
        if (t < C) {                                // everybody learns how many candidates everybody has, the first CTA the sums, too
            double sum = 0.0;
            for (int i = 0; i < F::WARPS; ++i) sum += sh.red[i];
            cluster_store_u32(&sh.peer_n[rank], t, (uint32_t)sh.n);
            cluster_store_f64(&sh.peer_sum[rank], t, sum);
            cluster_store_f64(&sh.peer_ref[rank], t, rest.far ? (double)INF_F : (double)rest.ref);
        }
        cluster_arrive_wait();
        const int n = sh.n;
        if (rank == 0) {
            // the sums, relative to the largest reference of those that have one
            float ref = -INF_F;
            for (int c = 0; c < C; ++c) {
                rest.far |= sh.peer_ref[c] == (double)INF_F;
                if (!(sh.peer_sum[c] == 0.0)) ref = fmaxf(ref, (float)sh.peer_ref[c]);
            }
            rest.s = 0.0f;
            rest.ref = ref;
            if (t < C && !(sh.peer_sum[t] == 0.0)) rest.s = (float)(sh.peer_sum[t] * (double)ex2((float)sh.peer_ref[t] - rest.ref));
        } else {
            int at = 0;
            for (int c = 0; c < rank; ++c) at += (int)sh.peer_n[c];
            for (int i = t; i < n; i += F::NT) cluster_store_u64(&sh.cand[at + i], 0, sh.cand[i]);
        }
        cluster_arrive_wait();
        if (rank != 0) return;
        if (t == 0) {
            int at = 0;
            for (int c = 0; c < C; ++c) at += (int)sh.peer_n[c];
            sh.n = at;
        }
        __syncthreads();
    }
    // in order: a few by the number of larger ones, many by a sorting network; what lies behind the k-th goes into the rest
    constexpr bool few = F::MOST_K <= 128;
    int most = 192;                                 // a network of k's power of two, not of a larger one: twice the size takes more than the bisection
    if (!few)
        for (most = 64; most < k;) most *= 2;
    if (sh.n > most) prune<T>(sh, k, few ? 64 : most - k, lo_key, K::MOST, rest);
    unsigned long long* cand = sh.cand;
    const int kept = sh.n;
    unsigned long long behind[few ? 1 : MAX_K / F::NT];
    if (few) {
        const unsigned long long mine = t < kept ? cand[t] : 0ull;
        if (t < 3) cand[kept + t] = 0ull;
        __syncthreads();
        int place = 0;
        if ((t & ~31) < kept) {
            const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(cand);
            int other = 0;
#pragma unroll 4
            for (int j = 0; j < (kept + 3) / 4; ++j) {
                const ulonglong2 p = pairs[2 * j], q = pairs[2 * j + 1];
                place += (int)(p.x > mine) + (int)(p.y > mine);
                other += (int)(q.x > mine) + (int)(q.y > mine);
            }
            place += other;
        }
        __syncthreads();
        if (t < kept && place < k) cand[place] = mine;
        __syncthreads();
        behind[0] = t < kept && place >= k ? mine : 0ull;
    } else {
        sort_descending<F>(cand, kept);
#pragma unroll
        for (int i = 0; i < (few ? 1 : MAX_K / F::NT); ++i) behind[i] = t + i * F::NT >= k && t + i * F::NT < kept ? cand[t + i * F::NT] : 0ull;
    }
    if (kept > k) {
        rest.move(K::bound((uint32_t)(cand[k - 1] >> 32)));
        double terms = 0.0;
#pragma unroll
        for (int i = 0; i < (few ? 1 : MAX_K / F::NT); ++i) if (behind[i]) terms += grid_term(rest, K::value_of(behind[i]));
        add_terms<F>(sh.terms, terms, rest);
    }
    for (int i = t; i < k; i += F::NT) {
        const unsigned long long c = cand[i];
        const int e = index_of(c);
        a.indices[row * k + i] = e;
        reinterpret_cast<T*>(a.values)[row * k + i] = g.p[e];
        if ((uint32_t)(c >> 32) == 0u) rest.s = K::value_of(c);             // a NaN in the list: the rest is NaN
    }
    float s = rest.s;
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane_id() == 0) sh.red[warp_id()] = (double)s;
    __syncthreads();
    double sum = 0.0;
    for (int i = 0; i < F::WARPS; ++i) sum += sh.red[i];
    double ref = (double)rest.ref * 0.69314718055994531;
    const unsigned long long last = cand[k - 1];
    if (a.vocab > k && (rest.far || (sum == sum && !(sum >= 1e-3)))) {
        // nothing to speak of relative to the bound (masked logits, a gap), or infinities: again, relative to the largest of the rest
        float m = -INF_F, bad = 0.0f;
        for (int e = t; e < a.vocab; e += F::NT) {
            const float x = Elem<T>::load(g.p, e);
            if (x != x) bad = x;
            else if (K::composite(x, e) < last) m = fmaxf(m, x);
        }
        const uint32_t top = __reduce_max_sync(0xffffffffu, ord_key(m));
        if (lane_id() == 0) sh.warp_max[warp_id()] = top;
        __syncthreads();
        m = -INF_F;
        for (int i = 0; i < F::WARPS; ++i) m = fmaxf(m, ord_value(sh.warp_max[i]));
        double part = (double)bad;
        if (m != -INF_F && m != INF_F)
            for (int e = t; e < a.vocab; e += F::NT) {
                const float x = Elem<T>::load(g.p, e);
                if (x == x && K::composite(x, e) < last) part += (double)ex2((x - m) * a.scale);
            }
#pragma unroll
        for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
        __syncthreads();
        if (lane_id() == 0) sh.red[warp_id()] = part;
        __syncthreads();
        sum = 0.0;
        for (int i = 0; i < F::WARPS; ++i) sum += sh.red[i];
        ref = m == -INF_F ? 0.0 : (double)m / a.tau;
        if (m == INF_F && sum == sum) sum = 1.0;
    }
    if (t == 0) a.rest[row] = sum == 0.0 ? -INF_F : (float)(ref + log(sum));
}

template <typename T, class F> int launch_form(Args a, int64_t rows, int sms, cudaStream_t s) {
    // CTAs of a row: until every SM has one, no part below 4 KB, and the merged lists fit the candidates' room
    a.cluster = 1;
    while (a.cluster < 8 && rows * a.cluster * 2 <= sms && (int64_t)a.vocab * sizeof(T) / (2 * a.cluster) >= 4096 && 2 * a.cluster * a.k <= F::CAP) a.cluster *= 2;
    // The sample: an eighth of a row of 128256 bf16 at least (2048 vectors), and so many that the list has room.  It holds k (part / sample) vectors, 1.3 to 1.5 times that
    // with the slack of the bound and groups of several, and for lists of any length varies by less than 1 / sqrt(k): 2 k (part / sample) fit.  In four times as many
    // groups as k, as far as the list's room goes.
    const int64_t part = ((int64_t)a.vocab / RowGrid<T>::N + a.cluster) / a.cluster;
    const int each = (int)std::max<int64_t>(2048 / F::NT, std::min<int64_t>(512, ceil_div64(2 * part * a.k, (int64_t)F::NT * F::LIST)));
    a.groups = std::min({F::LIST / F::NT, each, std::max(1, (4 * a.k + F::NT - 1) / F::NT)});
    a.per = (each + a.groups - 1) / a.groups;
    return launch_rows(topk_logits_kernel<T, F>, "topk_logits", rows * a.cluster, F::NT, sizeof(Shared<F>), a.cluster, s, a);
}

template <typename T> int launch(const Args& a, int64_t rows, cudaStream_t s) {
    const int sms = device_sm_count();
    if (sms < 0) return MAB_ERR_CUDA;
    return a.k <= Form<false>::MOST_K ? launch_form<T, Form<false>>(a, rows, sms, s) : launch_form<T, Form<true>>(a, rows, sms, s);
}

}  // namespace toplogits
}  // namespace mab

using namespace mab;

extern "C" int mab_topk_logits(int64_t rows, int64_t vocab, int64_t k, const void* logits, int dtype, int64_t pitch, double temperature,
                               void* values, int32_t* indices, float* rest, void* stream) {
    MAB_REQUIRE(rows >= 0 && vocab >= 1 && k >= 1 && k <= vocab, MAB_ERR_BAD_ARG, "mab_topk_logits: rows=%lld, vocab=%lld, k=%lld", (long long)rows,
                (long long)vocab, (long long)k);
    MAB_REQUIRE(dtype == MAB_F32 || dtype == MAB_BF16, MAB_ERR_UNSUPPORTED, "mab_topk_logits: element type %d", dtype);
    MAB_REQUIRE(temperature > 1e-6 && temperature < 1e6, MAB_ERR_BAD_ARG, "mab_topk_logits: temperature=%g outside (1e-6, 1e6)", temperature);
    MAB_REQUIRE(rows < (1 << 28) && vocab <= MAB_MAX_VOCAB && k <= MAB_MAX_LIST, MAB_ERR_LIMIT, "mab_topk_logits: rows=%lld, vocab=%lld, k=%lld beyond 2^28, %d, %d",
                (long long)rows, (long long)vocab, (long long)k, MAB_MAX_VOCAB, MAB_MAX_LIST);
    if (rows == 0) return MAB_OK;
    MAB_REQUIRE(logits && values && indices && rest, MAB_ERR_BAD_ARG, "mab_topk_logits: null pointer");
    MAB_REQUIRE(pitch >= vocab, MAB_ERR_BAD_ARG, "mab_topk_logits: rows of %lld logits lie %lld apart", (long long)vocab, (long long)pitch);
    const size_t e = dtype == MAB_F32 ? 4 : 2;
    MAB_REQUIRE(aligned_to(logits, e) && aligned_to(values, e) && aligned_to(indices, 4) && aligned_to(rest, 4), MAB_ERR_BAD_ARG, "mab_topk_logits: misaligned buffer");
    const Span in = {logits, rows, (int64_t)(vocab * e), (int64_t)(pitch * e)};
    const Span out[3] = {vector_span(values, rows * k * (int64_t)e), vector_span(indices, rows * k * 4), vector_span(rest, rows * 4)};
    MAB_REQUIRE(apart(in, out[0]) && apart(in, out[1]) && apart(in, out[2]) && apart(out[0], out[1]) && apart(out[0], out[2]) && apart(out[1], out[2]), MAB_ERR_BAD_ARG,
                "mab_topk_logits: the outputs overlap one another or the logits");
    toplogits::Args a = {};
    a.logits = logits; a.pitch = pitch; a.values = values; a.indices = indices; a.rest = rest; a.tau = temperature;
    a.scale = (float)(1.4426950408889634 / temperature); a.vocab = (int)vocab; a.k = (int)k;
    return dtype == MAB_F32 ? toplogits::launch<float>(a, rows, (cudaStream_t)stream) : toplogits::launch<uint16_t>(a, rows, (cudaStream_t)stream);
}
