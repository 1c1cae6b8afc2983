// out[i, j] = (sum_c a[i, c] b[j, c]) a_scale[i] b_scale[j] + bias[j]: 8-bit operands, exact 32-bit sums.
//
// The tensor cores' rows (128 lanes of tensor memory) are output channels (rows of b), their columns tokens (rows of a): a few tokens are a
// narrow tile, not a nearly empty one, and a warp of the epilogue holds 32 neighbouring channels of one token, so its stores are runs of 64 or 128 bytes without a
// detour through shared memory.  One warp issues tiled copies (128 bytes of the inner size, 128-byte swizzle, zeros beyond the edges) into a ring of
// stages, another the products, the others take the sums out of tensor memory.  Three forms, by the number of tokens (us, B200; here and in the other kernels of rows: a call in a row of calls
// from a graph, several sets of inputs in turn, so without the host):
//
// * up to 2 (4 where the weights are few): no tile at all, a warp per pair of channels, four products an instruction.  Bound by the weights' bytes: 4096 x 4096 3.4 for one token, 5.2 for
//   four (the tiles from 5 tokens on: 5.5).
// * up to 64: tiles of at most 128 channels and all tokens; where there are fewer tiles than SMs the inner size is split over the CTAs of a cluster, whose partial
//   sums meet in distributed shared memory: integers, so in any order the same.  Bound by the weights' bytes and some 5 us before the first and behind the last of them:
//   41 tokens, 14336 x 4096: 14.4 (59 MB); 16 tokens, 128256 x 4096: 80.5 (6.5 TB/s). (So, too, up to 128 where the channels are few and the inner size long.)
// * more: tiles of two CTAs.  Bound by the tensor cores where the inner size is long: 2048 tokens, 128256 x 4096: 640 to 800 by the state of the power cap (3.4 to 2.7
//   PFLOP/s, tensor pipe 98.4 % active); 4096^3: 46.3 (2.97); by the stores where it is short, an SM takes some 7 cycles for each 128-byte line that a warp stores to: 768 tokens,
//   50304 x 768 bf16 33, 777 tokens, 50257 x 767 fp32, where every run of 128 bytes touches two lines, 51 (the stores alone 46; 57 to 59 with outputs that were not in L2), 2048 tokens,
//   50257 x 768 fp32 152.  Rows through shared memory and bulk copies, from tiles that overlap by 16 bytes, took 53, and 114 for the 2048: not in the code, and the border between them not measured.
#include "rows.cuh"
#include "tcgen05.cuh"

namespace mab {
namespace int8mm {

constexpr int BM = 128, BK = 128;                  // channels of a tile, bytes of the inner size of a stage
constexpr int THREADS = 192;
__device__ int g_timeout;

struct Args {
    const int8_t *a, *b;
    int64_t a_pitch, b_pitch, out_pitch;
    const float *a_scales, *b_scales, *bias;
    void* out;
    int m, n, k;
    int token_tiles, split, stages, height;        // tiles of `height` channels (a multiple of 8, at most 128)
    int give_up;                                   // nothing is copied, as if every wait for it had run out (the selftest)
};
constexpr uint32_t NOT_A_NUMBER = 0x7FC00000u;     // the scale of the channels of a tile whose products did not come

__device__ __forceinline__ float scaled(int sum, float token, float channel, float bias) { return fmaf((float)sum * token, channel, bias); }

constexpr int MOST_STAGES = 9, RING_ONE = 200 * 1024, RING_TWO = 108 * 1024;      // the ring of one CTA, or of each of two, on an SM

template <typename T, int BN>
__global__ void __launch_bounds__(THREADS) int8_matmul_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                              const __grid_constant__ Args g) {
    constexpr int STAGE = (BM + BN) * BK;
    extern __shared__ unsigned char dyn[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[MOST_STAGES], empty[MOST_STAGES], done;
    __shared__ uint32_t s_tmem;
    __shared__ int s_lost;
    __shared__ float s_token[BN];
    __shared__ float2 s_channel[BM];
    constexpr uint32_t COLUMNS = BN < 32 ? 32 : BN;
    const int warp = warp_id(), lane = lane_id(), t = threadIdx.x;
    const int rank = g.split > 1 ? (int)(blockIdx.x % g.split) : 0;
    const int tile = blockIdx.x / g.split, token0 = tile % g.token_tiles * BN, channel0 = tile / g.token_tiles * g.height;
    const int steps = (g.k + BK - 1) / BK, k0 = (int)((int64_t)steps * rank / g.split), k1 = g.give_up ? k0 : (int)((int64_t)steps * (rank + 1) / g.split);
    const int stages = g.stages;
    auto load = [&](int i, int s) {                 // step i into stage s
        unsigned char* stage = ring + s * STAGE;
        mbar_arrive_expect_tx(&full[s], (uint32_t)(g.height + BN) * BK);
        tile_g2s(stage, &map_b, i * BK, channel0, &full[s]);
        tile_g2s(stage + BM * BK, &map_a, i * BK, token0, &full[s]);
    };
    if (t == 0) {
        for (int i = 0; i < stages; ++i) { mbar_init_unfenced(&full[i], 1); mbar_init_unfenced(&empty[i], 1); }
        mbar_init_unfenced(&done, 1);
        mbar_init_fence();
        s_lost = g.give_up;
    }
    if (warp == 1) tmem_alloc(&s_tmem, COLUMNS);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    // The next kernel begins not before this CTA has its tensor memory: a CTA of it that came first could hold all of it (the pairs take 512 columns) while it waits for this kernel.
    kernel_before_is_done();
    const uint32_t acc = s_tmem;
    if (t == 0)
        for (int i = k0; i < k1 && i < k0 + stages; ++i) load(i, i - k0);
    for (int i = t; i < BN; i += THREADS) s_token[i] = token0 + i < g.m ? g.a_scales[token0 + i] : 0.0f;
    if (t < BM) {
        const int channel = channel0 + t;
        s_channel[t] = t < g.height && channel < g.n ? make_float2(g.b_scales[channel], g.bias ? g.bias[channel] : 0.0f) : make_float2(0.0f, 0.0f);
    }

    if (warp < 2) {
        const bool issuing = elect_one();
        int s = 0;
        uint32_t parity = 0;
        auto next = [&] { if (++s == stages) { s = 0; parity ^= 1; } };
        if (warp == 0) {
            for (int i = k0 + stages; i < k1; ++i, next()) {
                if (!mbar_wait(&empty[s], parity)) { s_lost = 1; break; }
                if (issuing) load(i, s);
                __syncwarp();
            }
        } else {
            const uint32_t ring0 = smem_addr(ring);
            int i = k0;
            for (; i < k1; ++i, next()) {
                if (!mbar_wait(&full[s], parity)) { s_lost = 1; break; }
                tmem_fence_after();
                const uint32_t stage = ring0 + s * STAGE;
                const uint64_t wd = operand_desc(stage), td = operand_desc(stage + BM * BK);
                if (issuing) {
#pragma unroll
                    for (int j = 0; j < BK / 32; ++j) mma_i8(acc, wd + 2 * j, td + 2 * j, i8_instruction(BM, BN), i > k0 || j > 0);
                    mma_commit(&empty[s]);
                }
                __syncwarp();
            }
            const bool issued = i > k0;
            for (int n = 0; i < k1 && n < stages; ++i, ++n, next()) mbar_wait(&full[s], parity);      // lost: copies still on their way must not outlive the CTA
            if (issuing) {
                if (issued) mma_commit(&done);
                else mbar_arrive(&done);
            }
        }
    }
    __syncwarp();
    if (!mbar_wait(&done, 0)) atomicExch(&s_lost, 1);
    tmem_fence_after();
    __syncthreads();
    const bool lost = s_lost != 0;
    if (lost && t == 0) atomicExch(&g_timeout, 1);
    T* out = reinterpret_cast<T*>(g.out);

    if (g.split == 1) {
        if (warp >= 2) {
            const int quarter = warp & 3, at = 32 * quarter + lane, channel = channel0 + at;
            const bool there = at < g.height && channel < g.n;
            const float cs = lost ? __uint_as_float(NOT_A_NUMBER) : s_channel[at].x, bias = s_channel[at].y;
            for (int c = 0; c < BN && token0 + c < g.m; c += 16) {
                int r[16];
                tmem_load(acc + ((uint32_t)(32 * quarter) << 16) + c, r);
                tmem_wait_load(r);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (there && token0 + c + i < g.m)
                        Elem<T>::store(out, (int64_t)(token0 + c + i) * g.out_pitch + channel, scaled(r[i], s_token[c + i], cs, bias));
            }
        }
    } else {
        // the cluster's partial sums, [column][channel] in the ring, which every copy and product has left
        int* part = reinterpret_cast<int*>(ring);
        if (warp >= 2 && !lost) {
            const int quarter = warp & 3;
            for (int c = 0; c < BN; c += 16) {
                int r[16];
                tmem_load(acc + ((uint32_t)(32 * quarter) << 16) + c, r);
                tmem_wait_load(r);
#pragma unroll
                for (int i = 0; i < 16; ++i) part[(c + i) * BM + 32 * quarter + lane] = r[i];
            }
        }
        cluster_arrive_wait();
        const int there = min(BN, g.m - token0), c0 = there * rank / g.split, c1 = there * (rank + 1) / g.split;      // this CTA's columns
        bool any = false;
        for (int s = 0; s < g.split; ++s) any |= cluster_load_u32(&s_lost, s) != 0;
        if (any) {
            __syncthreads();
            if (t < BM) s_channel[t].x = __uint_as_float(NOT_A_NUMBER);
            __syncthreads();
        }
        for (int i = c0 * (BM / 4) + t; i < c1 * (BM / 4); i += THREADS) {
            const int column = i / (BM / 4), at = i % (BM / 4) * 4, channel = channel0 + at;
            int4 p[8], sum = make_int4(0, 0, 0, 0);
#pragma unroll
            for (int s = 0; s < 8; ++s) if (s < g.split) p[s] = cluster_load_int4(&part[4 * i], s);
#pragma unroll
            for (int s = 0; s < 8; ++s) if (s < g.split) { sum.x += p[s].x; sum.y += p[s].y; sum.z += p[s].z; sum.w += p[s].w; }
            const int sums[4] = {sum.x, sum.y, sum.z, sum.w};
            T* o = out + (int64_t)(token0 + column) * g.out_pitch + channel;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (at + j < g.height && channel + j < g.n)
                    Elem<T>::store(o, j, scaled(sums[j], s_token[column], s_channel[at + j].x, s_channel[at + j].y));
        }
        cluster_arrive_wait();
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 1) { tmem_fence_after(); tmem_free(acc, COLUMNS); }
}

// A wait that runs out (a device in trouble) sets the library's flag, and the tiles concerned are NaN.
//
// The form for many tokens: two CTAs share a tile of 256 channels and up to 256 tokens, so a stage of the ring is 16 KB of weights and up to 16 KB of tokens
// a CTA for twice the products, and they stay on their SMs: while other warps take the sums of one tile out of tensor memory, the next tile's go into its other
// half.  Tiles of the same channels follow one another: the weights come from HBM once.
constexpr int PAIR_SLICES = 2, PAIR_WARPS = 4 * PAIR_SLICES, PAIR_THREADS = 32 * (2 + PAIR_WARPS);
constexpr int PAIR_STAGES = 6, PAIR_STAGE = 2 * BM * BK, PAIR_LIMIT = 1 << 18;
constexpr int PAIR_BYTES = PAIR_STAGE * PAIR_STAGES + 1024;

template <typename T>
__global__ void __launch_bounds__(PAIR_THREADS) int8_matmul_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                                        const __grid_constant__ Args g, int tokens, int tiles) {
    extern __shared__ unsigned char dyn[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[PAIR_STAGES], empty[PAIR_STAGES], ready[2], taken[2], drained;
    __shared__ uint32_t s_tmem;
    __shared__ int s_lost;
    const int warp = warp_id(), lane = lane_id(), t = threadIdx.x, rank = (int)(blockIdx.x & 1), pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);
    const int steps = (g.k + BK - 1) / BK;
    if (t == 0) {
        for (int i = 0; i < PAIR_STAGES; ++i) { mbar_init_unfenced(&full[i], 1); mbar_init_unfenced(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init_unfenced(&ready[i], 1); mbar_init_unfenced(&taken[i], 2 * PAIR_WARPS); }
        mbar_init_unfenced(&drained, 1);
        mbar_init_fence();
        s_lost = 0;
    }
    if (warp == 1) tmem_alloc_pair(&s_tmem, 512);
    tmem_fence_before();
    __syncthreads();
    cluster_arrive_wait();                          // the other CTA's barriers are there
    tmem_fence_after();
    kernel_before_is_done();
    const uint32_t acc = s_tmem;

    if (warp < 2) {
        const bool issuing = elect_one();
        int s = 0;
        uint32_t parity = 0;
        auto next = [&] { if (++s == PAIR_STAGES) { s = 0; parity ^= 1; } };
        bool ok = !g.give_up;
        if (warp == 0) {
            const uint32_t full0 = cluster_addr(&full[0], 0), bytes = (uint32_t)(2 * BM + tokens) * BK;       // both CTAs' bytes
            int filled = 0;
            for (int tile = pair; ok && tile < tiles; tile += pairs) {
                const int token0 = tile % g.token_tiles * tokens + rank * (tokens / 2), channel0 = tile / g.token_tiles * 2 * BM + rank * BM;
                for (int i = 0; i < steps; ++i, next()) {
                    if (filled == PAIR_STAGES) {
                        if (!mbar_wait(&empty[s], parity ^ 1, PAIR_LIMIT)) { ok = false; break; }
                    } else {
                        ++filled;
                    }
                    if (issuing) {
                        unsigned char* stage = ring + s * PAIR_STAGE;
                        const uint32_t bar = full0 + 8 * s;
                        if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
                        tile_g2s_pair(stage, &map_b, i * BK, channel0, bar);
                        tile_g2s_pair(stage + BM * BK, &map_a, i * BK, token0, bar);
                    }
                    __syncwarp();
                }
            }
        } else if (rank == 0) {
            const uint32_t instruction = i8_instruction(2 * BM, tokens), ring0 = smem_addr(ring);
            int done = 0;                           // tiles
            const int64_t total = ok ? (int64_t)((tiles - pair + pairs - 1) / pairs) * steps : 0;       // stages' fillings
            int64_t left = total;                   // ... that have not been waited for
            for (int tile = pair; ok && tile < tiles; tile += pairs, ++done) {
                const uint32_t d = acc + (done & 1) * 256;
                if (done >= 2 && !mbar_wait(&taken[done & 1], (done / 2 - 1) & 1, PAIR_LIMIT)) { ok = false; break; }
                tmem_fence_after();
                for (int i = 0; i < steps; ++i, --left, next()) {
                    if (!mbar_wait(&full[s], parity, PAIR_LIMIT)) { ok = false; break; }
                    tmem_fence_after();
                    const uint32_t stage = ring0 + s * PAIR_STAGE;
                    const uint64_t wd = operand_desc(stage), td = operand_desc(stage + BM * BK);
                    if (issuing) {
#pragma unroll
                        for (int j = 0; j < BK / 32; ++j) mma_i8_pair(d, wd + 2 * j, td + 2 * j, instruction, i > 0 || j > 0);
                        mma_commit_pair(&empty[s]);
                    }
                    __syncwarp();
                }
                if (ok && issuing) mma_commit_pair(&ready[done & 1]);
                __syncwarp();
            }
            if (!ok) {                              // copies and products that may still be on their way must not outlive the CTAs
                const bool issued = left < total;
                for (int i = 0; i < PAIR_STAGES && i < left; ++i, next()) mbar_wait(&full[s], parity, PAIR_LIMIT);
                if (issued) {
                    if (issuing) mma_commit_pair(&drained, 1);
                    __syncwarp();
                    mbar_wait(&drained, 0, PAIR_LIMIT);
                }
            }
        }
        if (!ok) s_lost = 1;
    } else {
        // 32 channels and every other group of 32 tokens a warp
        const int quarter = warp & 3, slice = (warp - 2) >> 2, groups = tokens / 32;
        int done = 0;
        bool lost = g.give_up;                      // (from there on every tile of the pair is NaN)
        for (int tile = pair; tile < tiles; tile += pairs, ++done) {
            const int token0 = tile % g.token_tiles * tokens, channel = tile / g.token_tiles * 2 * BM + rank * BM + 32 * quarter + lane;
            const bool there = channel < g.n;
            float cs = there ? g.b_scales[channel] : 0.0f;
            const float bias = g.bias && there ? g.bias[channel] : 0.0f;
            auto scale_of = [&](int group) {          // of the group's tokens, one a lane
                const int token = token0 + 32 * group + lane;
                return group < groups && token < g.m ? g.a_scales[token] : 0.0f;
            };
            float next_scale = scale_of(slice);
            if (lost || !mbar_wait(&ready[done & 1], done / 2 & 1, PAIR_LIMIT)) {
                lost = true;
                s_lost = 1;
                cs = __uint_as_float(NOT_A_NUMBER);
            }
            __syncwarp();
            tmem_fence_after();
            const uint32_t from = acc + ((uint32_t)(32 * quarter) << 16) + (done & 1) * 256;
            if (slice >= groups && lane == 0) mbar_arrive_cluster(cluster_addr(&taken[done & 1], 0));
            // not unrolled: a tile's instructions would not fit the cache (768 tokens, 50304 x 768 bf16 36 us, 777, 50257 x 767 fp32 59; rolled and with one way for whole and partial groups 33 and 50)
#pragma unroll 1
            for (int group = slice; group < groups; group += PAIR_SLICES) {
                int r[32];
                tmem_load(from + 32 * group, r);
                const float scale = next_scale;
                next_scale = scale_of(group + PAIR_SLICES);
                tmem_wait_load(r);
                if (group + PAIR_SLICES >= groups) {          // the warp's sums of the tile are in registers
                    tmem_fence_before();
                    if (lane == 0) mbar_arrive_cluster(cluster_addr(&taken[done & 1], 0));
                }
                const int first = token0 + 32 * group, there_tokens = g.m - first;
                T* out = reinterpret_cast<T*>(g.out) + (int64_t)first * g.out_pitch + channel;
#pragma unroll
                for (int i = 0; i < 32; ++i, out += g.out_pitch) {
                    const float s = __shfl_sync(0xffffffffu, scale, i);
                    if (there && i < there_tokens) Elem<T>::store(out, 0, scaled(r[i], s, cs, bias));
                }
            }
        }
    }
    __syncwarp();
    tmem_fence_before();
    __syncthreads();
    if (s_lost && t == 0) atomicExch(&g_timeout, 1);
    cluster_arrive_wait();                          // nobody reports to a CTA that is gone
    tmem_fence_after();
    if (warp == 1) tmem_free_pair(acc, 512);
}

// 16 codes, by a load that the compiler leaves where it is: the kernel before, which may have written them, was still running when this one began, so they are neither the non-coherent
// path's (for what nobody writes meanwhile) nor to be asked for before the wait; and all of a round's are on their way together (4 tokens, 4096 x 14336: 24.2 us by plain C++ loads, 19.5).
__device__ __forceinline__ int4 load_codes(const int8_t* p) {
    int4 r;
    asm volatile("ld.global.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p) : "memory");
    return r;
}

// M tokens (m of them there): a warp for R channels, its lanes over the inner size.
template <typename T, int M, int R>
__global__ void __launch_bounds__(256) int8_rows_kernel(const __grid_constant__ Args g) {
    const int lane = lane_id(), channel0 = (blockIdx.x * 8 + warp_id()) * R;
    kernel_before_is_done();
    if (channel0 >= g.n) return;
    int acc[M][R];
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[i][r] = 0;
    const int8_t* b[R];
    const int8_t* a[M];
#pragma unroll
    for (int r = 0; r < R; ++r) b[r] = g.b + (int64_t)min(channel0 + r, g.n - 1) * g.b_pitch;
#pragma unroll
    for (int i = 0; i < M; ++i) a[i] = g.a + (int64_t)min(i, g.m - 1) * g.a_pitch;
    const int whole = g.k / 16;
#pragma unroll 4
    for (int v = lane; v < whole; v += 32) {
        int4 w[R];
#pragma unroll
        for (int r = 0; r < R; ++r) w[r] = load_codes(b[r] + 16 * v);
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int4 x = load_codes(a[i] + 16 * v);
#pragma unroll
            for (int r = 0; r < R; ++r)
                acc[i][r] = __dp4a(x.x, w[r].x, __dp4a(x.y, w[r].y, __dp4a(x.z, w[r].z, __dp4a(x.w, w[r].w, acc[i][r]))));
        }
    }
    const int c = whole * 16 + lane;                // the last, partial vector by bytes
    if (lane < 16 && c < g.k)
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
            for (int r = 0; r < R; ++r) acc[i][r] += (int)a[i][c] * (int)b[r][c];
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[i][r] = __reduce_add_sync(0xffffffffu, acc[i][r]);
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (lane == i * R + r && i < g.m && channel0 + r < g.n)
                Elem<T>::store(reinterpret_cast<T*>(g.out), (int64_t)i * g.out_pitch + channel0 + r,
                               scaled(acc[i][r], g.a_scales[i], g.b_scales[channel0 + r], g.bias ? g.bias[channel0 + r] : 0.0f));
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// Rows of k bytes, `pitch` apart, in boxes of box_rows x 128 bytes.
static int make_map(CUtensorMap* map, const int8_t* p, int64_t rows, int64_t k, int64_t pitch, int box_rows) {
    const EncodeTiled fn = encode_tiled();
    MAB_REQUIRE(fn, MAB_ERR_CUDA, "cuTensorMapEncodeTiled is not in this driver");
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2] = {BK, (cuuint32_t)box_rows}, ones[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    MAB_REQUIRE(r == CUDA_SUCCESS, MAB_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
    return MAB_OK;
}

// Tiles of at most 128 channels for all tokens; where those are fewer than the SMs, the inner size split over 2, 4 or 8 CTAs.  The height of the tiles and the split
// are those by which the SM with the most has the least to load.
template <typename T, int BN> int launch_tiles(Args g, int sms, cudaStream_t s) {
    const int steps = (g.k + BK - 1) / BK;
    g.token_tiles = (g.m + BN - 1) / BN;
    int64_t best = INT64_MAX;
    for (int split = 1; split <= 8 && (split == 1 || steps >= 2 * split); split *= 2)
        for (int height = BM; height >= 64; height -= 8) {
            const int64_t tiles = (int64_t)g.token_tiles * ceil_div64(g.n, height);
            const int64_t load = ceil_div64(tiles * split, split > 2 ? sms - sms / 8 : sms) * ((int64_t)ceil_div64(steps, split) * (height + BN) + 128 * (split > 1));
            if (load < best) { best = load; g.split = split; g.height = height; }
        }
    const int64_t ctas = (int64_t)g.token_tiles * ceil_div64(g.n, g.height) * g.split;
    const int stage = (BM + BN) * BK, most = (ctas > sms || g.split > 1 ? RING_TWO : RING_ONE) / stage;
    const int sums = g.split > 1 ? BM * BN * 4 : 0;                        // the partial sums have to fit the ring
    g.stages = std::max({1, std::min({most, MOST_STAGES, (steps + g.split - 1) / g.split}), (sums + stage - 1) / stage});
    CUtensorMap map_a, map_b;
    if (int rc = make_map(&map_a, g.a, g.m, g.k, g.a_pitch, BN)) return rc;
    if (int rc = make_map(&map_b, g.b, g.n, g.k, g.b_pitch, g.height)) return rc;
    return launch_rows(int8_matmul_kernel<T, BN>, "int8_matmul", ctas, THREADS, (size_t)stage * g.stages + 1024, g.split, s, map_a, map_b, g);
}

// Tiles of 256 channels and a multiple of 32 tokens, as many tokens as give the shortest time: a step of the inner size takes tokens x 2 cycles of products or
// the loading of 16 KB of weights and the tokens at some 50 bytes a cycle, whichever is more; the epilogue is seen once, after the last tile.
template <typename T> int launch_pairs(Args g, int sms, cudaStream_t s) {
    const int steps = (g.k + BK - 1) / BK, channel_tiles = (g.n + 2 * BM - 1) / (2 * BM);
    int tokens = 256;
    double best = 1e300;
    for (int parts = (g.m + 255) / 256, n = 0; n < 8; ++n, ++parts) {
        const int each = ((g.m + parts - 1) / parts + 31) / 32 * 32;
        const double waves = (double)ceil_div64((int64_t)ceil_div64(g.m, each) * channel_tiles, sms / 2);
        const double step = std::max(2.0 * each, (BM + each / 2) * BK / 50.0), epilogue = 2500 + 24.0 * each;
        const double time = waves * std::max(steps * step, epilogue) + epilogue;
        if (time < best * 0.98) { best = time; tokens = each; }
        if (each == 32) break;
    }
    CUtensorMap map_a, map_b;
    if (int rc = make_map(&map_a, g.a, g.m, g.k, g.a_pitch, tokens / 2)) return rc;
    if (int rc = make_map(&map_b, g.b, g.n, g.k, g.b_pitch, BM)) return rc;
    g.token_tiles = (g.m + tokens - 1) / tokens;
    const int64_t tiles = (int64_t)g.token_tiles * ((g.n + 2 * BM - 1) / (2 * BM));
    const int64_t pairs = std::min<int64_t>(tiles, sms / 2);
    return launch_rows(int8_matmul_pair_kernel<T>, "int8_matmul", pairs * 2, PAIR_THREADS, PAIR_BYTES, 2, s, map_a, map_b, g, tokens, (int)tiles);
}

// Tokens without a tile: one and two, and up to four where the weights are no more than 16 MB.  us, without and with: 4 x 1000 x 512 2.25 and 3.75, 4 x 4096 x 4096 5.2 and 5.45,
// 4 x 20000 x 1000 7.95 and 7.3, 3 x 14336 x 4096 19.3 and 12.8, 4 x 128256 x 4096 120 and 78; one token of 128256 x 4096 takes 79 without.
static bool without_tile(int64_t m, int64_t n, int64_t k) { return m <= 2 || (m <= 4 && n * k <= 1 << 24); }

template <typename T> int launch(const Args& g, cudaStream_t s) {
    const int sms = device_sm_count();
    if (sms < 0) return MAB_ERR_CUDA;
    if (without_tile(g.m, g.n, g.k)) {
        const int64_t ctas = ceil_div64(g.n, 16);
        if (g.m == 1) return launch_rows(int8_rows_kernel<T, 1, 2>, "int8_matmul", ctas, 256, 0, 1, s, g);
        if (g.m == 2) return launch_rows(int8_rows_kernel<T, 2, 2>, "int8_matmul", ctas, 256, 0, 1, s, g);
        return launch_rows(int8_rows_kernel<T, 4, 2>, "int8_matmul", ctas, 256, 0, 1, s, g);
    }
    // Few channels and a long inner size leave most SMs without a pair's tile: 65 and 128 tokens, 4096 x 14336, 25 us, in tiles with the inner size split 17.5 and 19 (with an
    // inner size of 4096 9.3 and 9.8 against 7.5 and 8.9, of 2048 6.3 and 6.7 against 6.6 and 8.0).
    if (g.m > 64 && g.m <= 128 && g.k > 48 * BK && 8 * ceil_div64(g.n, 2 * BM) <= sms) return launch_tiles<T, 128>(g, sms, s);
    if (g.m > 64) return launch_pairs<T>(g, sms, s);
    if (g.m <= 16) return launch_tiles<T, 16>(g, sms, s);
    if (g.m <= 32) return launch_tiles<T, 32>(g, sms, s);
    return launch_tiles<T, 64>(g, sms, s);
}

}  // namespace int8mm

int copy_timeout_int8_matmul(int* out, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(out, int8mm::g_timeout, sizeof(int));
    if (e == cudaSuccess && clear) { const int z = 0; e = cudaMemcpyToSymbol(int8mm::g_timeout, &z, sizeof(int)); }
    return e == cudaSuccess ? MAB_OK : cuda_fail(e, "int8_matmul wait flag");
}

}  // namespace mab

using namespace mab;

static int int8_matmul(int give_up, int64_t m, int64_t n, int64_t k, const int8_t* a, int64_t a_pitch, const int8_t* b, int64_t b_pitch,
                               const float* a_scales, const float* b_scales, const float* bias, void* out, int out_dtype, int64_t out_pitch,
                               void* stream) {
    MAB_REQUIRE(m >= 0 && n >= 0 && k >= 1, MAB_ERR_BAD_ARG, "mab_int8_matmul: m=%lld, n=%lld, k=%lld", (long long)m, (long long)n, (long long)k);
    MAB_REQUIRE(out_dtype == MAB_F32 || out_dtype == MAB_BF16, MAB_ERR_UNSUPPORTED, "mab_int8_matmul: element type %d", out_dtype);
    MAB_REQUIRE(m < (1 << 30) && n < (1 << 30) && k <= MAB_MAX_INNER && ceil_div64(m, 16) * ceil_div64(n, 128) < (1 << 28), MAB_ERR_LIMIT,
                "mab_int8_matmul: m=%lld, n=%lld, k=%lld (at most %d)", (long long)m, (long long)n, (long long)k, MAB_MAX_INNER);
    if (m == 0 || n == 0) return MAB_OK;
    MAB_REQUIRE(a && b && a_scales && b_scales && out, MAB_ERR_BAD_ARG, "mab_int8_matmul: null pointer");
    MAB_REQUIRE(a_pitch >= k && b_pitch >= k && out_pitch >= n, MAB_ERR_BAD_ARG, "mab_int8_matmul: rows lie %lld, %lld, %lld apart", (long long)a_pitch,
                (long long)b_pitch, (long long)out_pitch);
    MAB_REQUIRE(aligned_to(a, 16) && aligned_to(b, 16) && a_pitch % 16 == 0 && b_pitch % 16 == 0, MAB_ERR_BAD_ARG,
                "mab_int8_matmul: codes have to start on 16 bytes, their rows a multiple of 16 apart (%lld, %lld)", (long long)a_pitch, (long long)b_pitch);
    MAB_REQUIRE(aligned_to(a_scales, 4) && aligned_to(b_scales, 4) && aligned_to(bias, 4) && aligned_to(out, out_dtype == MAB_F32 ? 4 : 2),
                MAB_ERR_BAD_ARG, "mab_int8_matmul: misaligned buffer");
    const int64_t e = out_dtype == MAB_F32 ? 4 : 2;
    const Span to = {out, m, n * e, out_pitch * e};
    MAB_REQUIRE(apart(to, {a, m, k, a_pitch}) && apart(to, {b, n, k, b_pitch}) && apart(to, vector_span(a_scales, m * 4)) && apart(to, vector_span(b_scales, n * 4)) &&
                    apart(to, vector_span(bias, n * 4)), MAB_ERR_BAD_ARG, "mab_int8_matmul: out overlaps an operand, scales or the bias");
    int8mm::Args g = {a, b, a_pitch, b_pitch, out_pitch, a_scales, b_scales, bias, out, (int)m, (int)n, (int)k, 1, 1, 1, int8mm::BM, give_up};
    return out_dtype == MAB_F32 ? int8mm::launch<float>(g, (cudaStream_t)stream) : int8mm::launch<uint16_t>(g, (cudaStream_t)stream);
}

extern "C" int mab_int8_matmul(int64_t m, int64_t n, int64_t k, const int8_t* a, int64_t a_pitch, const int8_t* b, int64_t b_pitch,
                               const float* a_scales, const float* b_scales, const float* bias, void* out, int out_dtype, int64_t out_pitch,
                               void* stream) {
    return int8_matmul(0, m, n, k, a, a_pitch, b, b_pitch, a_scales, b_scales, bias, out, out_dtype, out_pitch, stream);
}

extern "C" int mab_int8_matmul_selftest(int64_t m, int64_t n, int64_t k, const int8_t* a, int64_t a_pitch, const int8_t* b,
                                        int64_t b_pitch, const float* a_scales, const float* b_scales, const float* bias, void* out, int out_dtype,
                                        int64_t out_pitch, void* stream) {
    return int8_matmul(1, m, n, k, a, a_pitch, b, b_pitch, a_scales, b_scales, bias, out, out_dtype, out_pitch, stream);
}
