// The k largest logits of every row, in descending order (ties: the lower index first), and rest = log sum exp(z / tau) over all others.
//
// One pass over the row.  The first chunk gives a bound: the k-th largest of its vectors' maxima, which at least k values reach.  From then on
// a value above the bound becomes a candidate in shared memory (some k ln(row / chunk) of a row do), every other one goes into the sum at once,
// relative to the bound, so the sum over the rest is its own and not a difference of two large ones.  When the candidates outgrow half of their room, the k
// largest of them stay, the others go into the sum, and the bound rises to the k-th; a chunk whose candidates do not fit (ascending rows, a
// chunk of one value) is selected from exactly, in registers.  At the end every candidate counts those before it, which is its place.
//
// The order is that of 64-bit keys, value above 2^32 - 1 - index: distinct, so "larger" contains the tie rule.  NaN lies below -inf and makes
// the rest NaN.  A row belongs to a cluster of one to eight CTAs; the first of them merges the candidates of all.
#include "rows.cuh"

namespace mab {
namespace toplogits {

constexpr int NT = 512, WARPS = NT / 32;
constexpr int UNROLL = 4;                          // vectors a thread holds of a chunk
constexpr int CAP = 4096;                          // candidates
constexpr int ROOM = CAP / 2;                      // pruned to k when more are there after a chunk
constexpr int MAX_K = 1024;
constexpr int ITEMS = CAP / NT;
constexpr int LAST = MAX_K / NT;                    // candidates a thread has in the end
static_assert(ROOM + MAX_K <= CAP && 8 * MAX_K / 2 <= CAP, "a chunk's exact selection and a merge have room");

struct Args {
    const void* logits;
    int64_t pitch;
    void* values;
    int32_t* indices;
    float* rest;
    double tau;
    float scale;
    int vocab, k, cluster;
};

struct Shared {
    unsigned long long cand[CAP];
    double red[WARPS];
    double sum;                                     // this CTA's sum over the rest, and its reference
    float ref;
    int n;                                          // candidates (can count beyond CAP while a chunk overflows)
    int count[64];                                  // counters of a bisection, one per step
    uint32_t warp_max[WARPS];
    int scan[40];
    unsigned long long kth;
};

// A thread's sum over the rest, relative to exp(ref).
struct Rest {
    float s, ref, scale;
    __device__ __forceinline__ void add(float x) { s += ex2((x - ref) * scale); }
    __device__ __forceinline__ void move(float to) {                                 // references only rise (from none: 0)
        if (to == -INF_F) to = 0.0f;
        if (!(s == 0.0f)) s *= ex2((ref - to) * scale);
        ref = to;
    }
};

__device__ __forceinline__ unsigned long long composite(float x, int e) { return (unsigned long long)row_key(x) << 32 | (0xFFFFFFFFu - (uint32_t)e); }
__device__ __forceinline__ int index_of(unsigned long long c) { return (int)(0xFFFFFFFFu - (uint32_t)c); }
__device__ __forceinline__ float value_of(unsigned long long c) { return ord_value((uint32_t)(c >> 32)); }

// Sum of one int per thread, step `i` of a bisection: counters are cleared by `clear_counts`, each is used once.
__device__ __forceinline__ int block_count(Shared& sh, int c, int i) {
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane_id() == 0 && c) atomicAdd(&sh.count[i], c);
    __syncthreads();
    return sh.count[i];
}
__device__ __forceinline__ void clear_counts(Shared& sh) {
    __syncthreads();
    if (threadIdx.x < 64) sh.count[threadIdx.x] = 0;
    __syncthreads();
}

// Largest key T with count(>= T) >= k, `counted(mid)` being the calling thread's number of keys >= mid.  Needs count(>= lo) >= k.
template <typename F> __device__ __forceinline__ uint32_t kth_key(Shared& sh, uint32_t lo, uint32_t hi, int k, F counted) {
    clear_counts(sh);
    for (int i = 0; lo < hi; ++i) {                 // invariant: count(>= lo) >= k, count(>= hi + 1) < k
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        if (block_count(sh, counted(mid), i) >= k) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// The k largest of the n > k candidates stay; the others go into the rest.  Returns the k-th key.
__device__ __noinline__ uint32_t prune(Shared& sh, int k, Rest& rest) {
    const int t = threadIdx.x, n = sh.n;
    unsigned long long c[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) c[i] = t + i * NT < n ? sh.cand[t + i * NT] : 0ull;
    auto there = [&](int i) { return t + i * NT < n; };
    const uint32_t T = kth_key(sh, 0u, 0xFFFFFFFFu, k, [&](uint32_t mid) {
        int r = 0;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) r += there(i) && (uint32_t)(c[i] >> 32) >= mid;
        return r;
    });
    clear_counts(sh);
    int above = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) above += there(i) && (uint32_t)(c[i] >> 32) > T;
    above = block_count(sh, above, 0);
    const uint32_t L = kth_key(sh, 0u, 0xFFFFFFFFu, k - above, [&](uint32_t mid) {      // among the equals: the largest low words (lowest indices)
        int r = 0;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) r += there(i) && (uint32_t)(c[i] >> 32) == T && (uint32_t)c[i] >= mid;
        return r;
    });
    const unsigned long long last = (unsigned long long)T << 32 | L;
    __syncthreads();
    if (t == 0) sh.n = 0;
    __syncthreads();
    rest.move(T > KEY_NEG_INF ? ord_value(T) : -INF_F);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if (!there(i)) continue;
        if (c[i] >= last) sh.cand[atomicAdd(&sh.n, 1)] = c[i];
        else rest.add(value_of(c[i]));
    }
    __syncthreads();
    return T;
}

template <typename T>
__global__ void __launch_bounds__(NT, 2) topk_logits_kernel(Args a) {
    constexpr int N = RowGrid<T>::N;
    extern __shared__ __align__(16) unsigned char dyn[];
    Shared& sh = *reinterpret_cast<Shared*>(dyn);
    const int C = a.cluster, rank = C > 1 ? (int)(blockIdx.x % C) : 0, t = threadIdx.x, k = a.k;
    const int64_t row = blockIdx.x / C;
    const RowGrid<T> g(reinterpret_cast<const T*>(a.logits) + row * a.pitch, a.vocab);
    const int per = (g.count + C - 1) / C, v0 = min(rank * per, g.count), v1 = min(v0 + per, g.count);
    if (t == 0) sh.n = 0;
    __syncthreads();
    Rest rest = {0.0f, 0.0f, a.scale};
    float bound = -INF_F;                           // values above it are candidates
    bool all = true;                                // no bound yet: everything is one, NaN too

    for (int base = v0; base < v1; base += NT * UNROLL) {
        // a chunk: the vectors base + u NT + t.  The partial vectors are among the first and the last; what lies outside the row has no place.
        uint4 raw[UNROLL];
        int e_first[UNROLL];
        uint32_t valid[UNROLL];                     // bits of the elements that are there
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int v = base + u * NT + t;
            valid[u] = 0;
            raw[u] = make_uint4(0, 0, 0, 0);
            e_first[u] = g.first(v);
            if (v < v1) {
                if (g.whole(v)) { raw[u] = g.load(v); valid[u] = (1u << N) - 1u; }
                else {
                    float x[N];
                    g.load_part(v, x, 0.0f);
                    raw[u] = pack(x, (const T*)nullptr);
#pragma unroll
                    for (int i = 0; i < N; ++i) if (e_first[u] + i >= 0 && e_first[u] + i < g.n) valid[u] |= 1u << i;
                }
            }
        }
        const int n0 = sh.n;
        const float s0 = rest.s;
        bool exact = false;
        if (all && min(v1 - base, NT * UNROLL) * N > ROOM) {
            // a bound that at least k values of this chunk reach: the k-th largest of the vectors' maxima
            uint32_t key[UNROLL];
            uint32_t top = 0;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                float x[N], m = -INF_F;
                unpack(raw[u], x, (const T*)nullptr);
#pragma unroll
                for (int i = 0; i < N; ++i) if (valid[u] >> i & 1u) m = fmaxf(m, x[i]);
                key[u] = valid[u] ? row_key(m) : 0u;
                top = max(top, key[u]);
            }
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane_id() == 0) sh.warp_max[warp_id()] = top;
            clear_counts(sh);
            for (int i = 0; i < WARPS; ++i) top = max(top, sh.warp_max[i]);
            auto counted = [&](uint32_t mid) {
                int r = 0;
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) r += key[u] >= mid;
                return r;
            };
            uint32_t lo = KEY_NEG_INF + 1, hi = top;
            if (hi > lo && block_count(sh, counted(lo), 0) >= k) {
                for (int i = 1; lo < hi; ++i) {
                    const uint32_t mid = lo + (hi - lo) / 2 + 1;
                    const int c = block_count(sh, counted(mid), i);
                    if (c >= k) { lo = mid; if (c <= k + k / 4) break; }
                    else hi = mid - 1;
                }
                bound = below_key(lo);
                all = false;
                rest.move(bound);
            } else {
                exact = true;                       // fewer than k numbers among the maxima
            }
        }
        __syncthreads();                            // n0 is read
        if (!exact) {
            bool over = false;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                float x[N];
                unpack(raw[u], x, (const T*)nullptr);
                float m = x[0];
#pragma unroll
                for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
                if (all || m > bound || valid[u] != (1u << N) - 1u) {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        if (!(valid[u] >> i & 1u)) { x[i] = -INF_F; continue; }
                        if (all || x[i] > bound) {
                            const int at = atomicAdd(&sh.n, 1);
                            if (at < CAP) sh.cand[at] = composite(x[i], e_first[u] + i);
                            over |= at >= ROOM;
                            x[i] = -INF_F;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < N; ++i) rest.add(x[i]);
            }
            if (!__syncthreads_or(over)) continue;
            if (sh.n <= CAP) {
                const uint32_t T_ = prune(sh, k, rest);
                bound = T_ > KEY_NEG_INF ? ord_value(T_) : -INF_F;
                all = false;
                continue;
            }
        }
        // exact selection from the chunk: its k largest eligible elements (all, where there are fewer) are candidates, the others go into the rest
        __syncthreads();
        if (t == 0) sh.n = n0;
        rest.s = s0;
        const uint32_t floor_key = all ? 0u : (bound == -INF_F ? KEY_NEG_INF : row_key(bound)) + 1u;     // eligible: key >= floor_key
        auto counted = [&](uint32_t mid) {
            int r = 0;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                float x[N];
                unpack(raw[u], x, (const T*)nullptr);
#pragma unroll
                for (int i = 0; i < N; ++i) r += (valid[u] >> i & 1u) && row_key(x[i]) >= mid;
            }
            return r;
        };
        clear_counts(sh);
        const int eligible = block_count(sh, counted(floor_key), 0);
        uint32_t kth = floor_key;
        int need = 0x7FFFFFFF;                      // equals of the k-th that are taken, in the order of their indices
        if (eligible > k) {
            kth = kth_key(sh, floor_key, 0xFFFFFFFFu, k, counted);
            clear_counts(sh);
            need = k - block_count(sh, kth == 0xFFFFFFFFu ? 0 : counted(kth + 1u), 0);
            rest.move(kth > KEY_NEG_INF ? ord_value(kth) : -INF_F);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            float x[N];
            unpack(raw[u], x, (const T*)nullptr);
            int equal = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) equal += (valid[u] >> i & 1u) && row_key(x[i]) == kth;
            int total = 0;
            int before = need == 0x7FFFFFFF ? 0 : block_exclusive_scan(equal, sh.scan, total);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!(valid[u] >> i & 1u)) continue;
                const uint32_t key = row_key(x[i]);
                const bool take = key > kth || (key == kth && (need == 0x7FFFFFFF || before++ < need));
                if (take) sh.cand[atomicAdd(&sh.n, 1)] = composite(x[i], e_first[u] + i);
                else rest.add(x[i]);
            }
            if (need != 0x7FFFFFFF) need = max(0, need - total);
            __syncthreads();
        }
        if (eligible > k) { bound = kth > KEY_NEG_INF ? ord_value(kth) : -INF_F; all = false; }
        __syncthreads();
        if (sh.n > ROOM) {                          // (n0 + k can be beyond it: the next chunk needs the room)
            const uint32_t T_ = prune(sh, k, rest);
            bound = T_ > KEY_NEG_INF ? ord_value(T_) : -INF_F;
            all = false;
        }
    }
    __syncthreads();
    if (C > 1 && sh.n > k) prune(sh, k, rest);

    if (C > 1) {                                    // the first CTA takes over the others' candidates and sums
        float s = rest.s;
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane_id() == 0) sh.red[warp_id()] = (double)s;
        __syncthreads();
        if (t == 0) {
            double sum = 0.0;
            for (int i = 0; i < WARPS; ++i) sum += sh.red[i];
            sh.sum = sum;
            sh.ref = rest.ref;
        }
        cluster_arrive_wait();
        if (rank == 0) {
            const int mine = sh.n;
            int at = mine;
            for (int c = 1; c < C; ++c) {
                const int n = (int)cluster_load_u32(&sh.n, c);
                for (int i = t; i < n; i += NT) sh.cand[at + i] = cluster_load_u64(&sh.cand[i], c);
                at += n;
            }
            __syncthreads();
            if (t == 0) sh.n = at;
            float ref = -INF_F;                     // the largest reference of those that have a sum
            for (int c = 0; c < C; ++c)
                if (!(cluster_load_f64(&sh.sum, c) == 0.0)) ref = fmaxf(ref, cluster_load_f32(&sh.ref, c));
            rest.move(ref);
            if (t == 0)
                for (int c = 1; c < C; ++c) {
                    const double sum = cluster_load_f64(&sh.sum, c);
                    if (!(sum == 0.0)) rest.s += (float)(sum * exp(((double)cluster_load_f32(&sh.ref, c) - (double)rest.ref) / a.tau));
                }
            __syncthreads();
        }
        cluster_arrive_wait();
        if (rank != 0) return;
    }
    if (sh.n > k && sh.n > NT) prune(sh, k, rest);

    // places: the number of larger candidates
    const int n = sh.n;
    unsigned long long mine[LAST];
    int place[LAST];
#pragma unroll
    for (int i = 0; i < LAST; ++i) {
        mine[i] = t + i * NT < n ? sh.cand[t + i * NT] : 0ull;
        place[i] = 0;
    }
    for (int j = 0; j < n; ++j) {
        const unsigned long long other = sh.cand[j];
#pragma unroll
        for (int i = 0; i < LAST; ++i) place[i] += other > mine[i];
    }
#pragma unroll
    for (int i = 0; i < LAST; ++i) {
        if (t + i * NT >= n || place[i] >= k) continue;
        const int e = index_of(mine[i]);
        a.indices[row * k + place[i]] = e;
        reinterpret_cast<T*>(a.values)[row * k + place[i]] = g.p[e];
        if (place[i] == k - 1) sh.kth = mine[i];
    }
    __syncthreads();
    const uint32_t kth = (uint32_t)(sh.kth >> 32);
    rest.move(kth > KEY_NEG_INF ? ord_value(kth) : -INF_F);
#pragma unroll
    for (int i = 0; i < LAST; ++i) {
        if (t + i * NT >= n) continue;
        const float x = value_of(mine[i]);
        if (place[i] >= k) rest.add(x);
        else if (x != x) rest.s = x;                // a NaN in the list: the rest is NaN
    }
    float s = rest.s;
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane_id() == 0) sh.red[warp_id()] = (double)s;
    __syncthreads();
    double sum = 0.0;
    for (int i = 0; i < WARPS; ++i) sum += sh.red[i];
    double ref = (double)rest.ref;
    if (sum == sum ? (!(sum >= 1e-20) && a.vocab > k) : rest.ref == INF_F) {
        // nothing to speak of relative to the bound (masked logits, a gap), or infinities: again, relative to the largest of the rest
        const unsigned long long last = sh.kth;
        float m = -INF_F, bad = 0.0f;
        for (int e = t; e < a.vocab; e += NT) {
            const float x = Elem<T>::load(g.p, e);
            if (x != x) bad = x;
            else if (composite(x, e) < last) m = fmaxf(m, x);
        }
        m = ord_value(__reduce_max_sync(0xffffffffu, ord_key(m)));
        if (lane_id() == 0) sh.warp_max[warp_id()] = ord_key(m);
        __syncthreads();
        for (int i = 0; i < WARPS; ++i) m = fmaxf(m, ord_value(sh.warp_max[i]));
        double part = (double)bad;
        if (m != -INF_F && m != INF_F)
            for (int e = t; e < a.vocab; e += NT) {
                const float x = Elem<T>::load(g.p, e);
                if (x == x && composite(x, e) < last) part += (double)ex2((x - m) * a.scale);
            }
#pragma unroll
        for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
        __syncthreads();
        if (lane_id() == 0) sh.red[warp_id()] = part;
        __syncthreads();
        sum = 0.0;
        for (int i = 0; i < WARPS; ++i) sum += sh.red[i];
        ref = (double)m;
        if (m == INF_F && sum == sum) { sum = 1.0; }
        if (m == -INF_F) ref = 0.0;
    }
    if (t == 0) a.rest[row] = sum == 0.0 ? -INF_F : (float)(ref / a.tau + log(sum));
}

template <typename T> int launch(Args a, int64_t rows, cudaStream_t s) {
    const int sms = device_sm_count();
    if (sms < 0) return MAB_ERR_CUDA;
    // CTAs of a row: until every SM has one, no part below 4 KB, and the merged lists fit the candidates' room
    a.cluster = 1;
    while (a.cluster < 8 && rows * a.cluster * 2 <= sms && (int64_t)a.vocab * sizeof(T) / (2 * a.cluster) >= 4096 && 2 * a.cluster * a.k <= CAP) a.cluster *= 2;
    return launch_rows(topk_logits_kernel<T>, "topk_logits", rows * a.cluster, NT, sizeof(Shared), a.cluster, s, a);
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
    toplogits::Args a = {};
    a.logits = logits; a.pitch = pitch; a.values = values; a.indices = indices; a.rest = rest; a.tau = temperature;
    a.scale = (float)(1.4426950408889634 / temperature); a.vocab = (int)vocab; a.k = (int)k;
    return dtype == MAB_F32 ? toplogits::launch<float>(a, rows, (cudaStream_t)stream) : toplogits::launch<uint16_t>(a, rows, (cudaStream_t)stream);
}
