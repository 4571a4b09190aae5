// Low-rank adapters beside a shared projection: y[m] += scale_i * B_i (A_i x[m]) for the adapter i of row m, the rows of a
// call in groups (groups.cuh).  No counterpart in the reference.  x is not quantized; A_i [rank][K] and B_i [N][rank] are
// fp32, fp16 or bf16 as the adapter was trained.
//
//   shrink: t = scale_i * A_i x, a cluster per tile of the plan's rows and 64 ranks; its CTAs divide K, and their sums meet in
//           shared memory, in order.
//   expand: y += B_i t.
// With few rows one launch does both; with many, shrink is a launch in front of the projection and expand one behind it.
// Both on mma.sync.m16n8k8 (tf32 operands, fp32 sums), the adapter's rows on the 16-row side and the call's rows on the
// 8-column side.  A tf32 operand keeps 11 bits: fp16 and bf16 weights are exact in one, an fp32 number is two (its first 11
// bits and the next 11), so that a product costs two MMAs, or four with fp32 weights, and is off by 2^-20 at most.  Outputs are off by 2e-7 to
// 5e-7 of their size in the 2-norm, about as an fp32 product's are (1e-7 to 2e-7).
// The order of k in an MMA is free as long as both operands have the same: a lane takes consecutive k of a row (8 of a piece
// of 32), so that fragments come straight from global memory in 16-byte loads.
//
// Bound by the bytes of x, A, B and y where there are many, and in front of that by dependent steps: plan, rows, K, the sums' meeting, columns.
// Measured, both products: 8 rows x 4096 x 4096, 8 bf16 adapters of rank 16 (2 MB) 6.0 us, 61 rows x 4096 x 11008, 40 fp16 ones of rank 64
// (65 MB) 23.2, 2048 rows x 4096 x 4096, 4 bf16 ones of rank 32 (34 MB of x, 67 of y) 38.7.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <atomic>

#include "groups.cuh"
#include "quant_pre.cuh"

namespace cg = cooperative_groups;

namespace q4fc {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kRankBlock = 64;   // ranks of a CTA in shrink
constexpr int kMostSlices = 8;   // CTAs of a cluster
constexpr int kMostRanks = 256;

// D(16x8) += A(16x8) * B(8x8)
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32_of_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// x = hi + lo, cut off to 11 bits each (which cannot overflow; an infinity leaves NaN)
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
__device__ __forceinline__ float number(float v) { return v; }
__device__ __forceinline__ float number(__half v) { return __half2float(v); }
__device__ __forceinline__ float number(__nv_bfloat16 v) { return __bfloat162float(v); }

// NV consecutive values (plain loads: behind pdl_wait_prior_grid() they stay there); VEC: in as wide loads as they allow, all there or (valid <= 0) none
template <int NV, bool VEC, typename T>
__device__ __forceinline__ void load_values(const T* p, int64_t valid, T (&v)[NV]) {
    if constexpr (VEC) {
        constexpr int kBytes = NV * (int)sizeof(T), kStep = kBytes < 16 ? kBytes : 16;
        static_assert(kStep == 8 || kStep == 16, "two or four words");
#pragma unroll
        for (int i = 0; i < kBytes / kStep; i++) {
            if constexpr (kStep == 16) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (valid > 0) w = reinterpret_cast<const uint4*>(p)[i];
                *reinterpret_cast<uint4*>(reinterpret_cast<char*>(v) + 16 * i) = w;
            } else {
                uint2 w = make_uint2(0, 0);
                if (valid > 0) w = reinterpret_cast<const uint2*>(p)[i];
                *reinterpret_cast<uint2*>(reinterpret_cast<char*>(v) + 8 * i) = w;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++) v[i] = i < (int)valid ? p[i] : T(0.0f);
    }
}

// four weights as the rows' operand, and what fp32 ones leave
template <typename T>
__device__ __forceinline__ void operand(T a, T b, T c, T d, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    const float f[4] = {number(a), number(b), number(c), number(d)};
#pragma unroll
    for (int i = 0; i < 4; i++)
        if constexpr (sizeof(T) == 4) split(f[i], hi[i], lo[i]);
        else hi[i] = __float_as_uint(f[i]), lo[i] = 0;
}
// sum += the products of sixteen terms.  An MMA cuts its sum off, always towards zero, so that a long chain of them shrinks.  So a chain is
// short: the products with a rest first, while the sum is 2^-11 of the others' size and its cuts too, then two MMAs of the first bits.  An
// addition, which rounds, joins it to the others.  (Chains over eight or nine pieces of 32 k, or over all of a warp's where warps and CTAs
// divide K, were off by 1.5e-6 to 8.6e-6, of positive terms by up to 2.4e-5; both products of 2048 rows x 4096 x 4096, rank 32, 37.5 us,
// so 38.2.  Rests and first bits in turn, chains of eight to sixteen: 4.5e-7 to 1.4e-6.)
template <typename T>
__device__ __forceinline__ void add_products(float (&sum)[4], const uint32_t (&wh)[2][4], const uint32_t (&wl)[2][4], const uint4 (&x)[2]) {
    float part[4];
    mma_tf32_of_zero(part, wh[0], x[0].z, x[0].w);
    mma_tf32(part, wh[1], x[1].z, x[1].w);
    if constexpr (sizeof(T) == 4)
#pragma unroll
        for (int j = 0; j < 2; j++) mma_tf32(part, wl[j], x[j].z, x[j].w), mma_tf32(part, wl[j], x[j].x, x[j].y);
    mma_tf32(part, wh[0], x[0].x, x[0].y);
    mma_tf32(part, wh[1], x[1].x, x[1].y);
#pragma unroll
    for (int i = 0; i < 4; i++) sum[i] += part[i];
}

// *y += (a, b): nothing comes back, L2 adds.  (One addition for each element: no order to depend on.)
__device__ __forceinline__ void add_to(float* y, float a, float b) {
    asm volatile("red.global.add.v2.f32 [%0], {%1, %2};" ::"l"(y), "f"(a), "f"(b) : "memory");
}

struct LoraArgs {
    const float* x;
    const void *a, *b;
    const float* scales;   // of the adapters, or null
    float* y;
    float* t;              // [place in the plan's order][rank]
    const int4* tiles;
    const int *tile_count, *order;
    int64_t rows, K, ldx, N, ldy, slice_k;
    int rank, n;
    const int* offsets;
};

// A_i x of eight rows and MB times 16 ranks, by one warp: pieces of 32 k from k0 on, `step` apart, up to k_end.  `x`: the row of lane (g, t)'s
// g, if `live`; `ranks`: of A that are there.  DEPTH: pieces at a time of up to 32 ranks.  acc[m][i]: rank m * 16 + 8 (i / 2) + g of row 2t + i % 2.
template <typename T, int MB, bool VEC, bool PAST_L1, int DEPTH>
__device__ __forceinline__ void shrink_rows(const float* x, bool live, const T* a, int ranks, int64_t K, int64_t k0, int64_t k_end, int64_t step,
                                            float (&acc)[MB][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    auto there = [&](int64_t k0) {  // this lane's values of a piece (VEC: whether there are any)
        const int64_t left = k_end - k0 - 8 * t;
        return VEC ? left : left < 8 ? left : 8;
    };
    // past L1, value by value: every fourth one from t on instead of eight in a row, so that loads share sectors
    auto load_few = [&](const auto* p, int left, auto& v) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (4 * i < left) v[i] = __ldcg(p + 4 * i);
            else v[i] = 0.0f;
    };
    auto load_x = [&](int64_t k0, float (&v)[8]) {
        if constexpr (PAST_L1) load_few(x + k0 + t, live ? (int)(k_end - k0 < 32 ? k_end - k0 : 32) - t : 0, v);
        else load_values<8, VEC>(x + k0 + 8 * t, live ? there(k0) : 0, v);
    };
    auto load_a = [&](int64_t k0, int m, T (&w)[2][8]) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = m * 16 + h * 8 + g;
            if constexpr (PAST_L1) load_few(a + (int64_t)r * K + k0 + t, r < ranks ? (int)(k_end - k0 < 32 ? k_end - k0 : 32) - t : 0, w[h]);
            else load_values<8, VEC>(a + (int64_t)r * K + k0 + 8 * t, r < ranks ? there(k0) : 0, w[h]);
        }
    };
    auto split_x = [&](const float (&v)[8], int j, uint4 (&s)[2]) {
#pragma unroll
        for (int i = 0; i < 2; i++) split(v[j + 2 * i], s[i].x, s[i].z), split(v[j + 2 * i + 1], s[i].y, s[i].w);
    };
    auto multiply = [&](int m, const T (&w)[2][8], int j, const uint4 (&s)[2]) {
        uint32_t wh[2][4], wl[2][4];
#pragma unroll
        for (int i = 0; i < 2; i++) operand(w[0][j + 2 * i], w[1][j + 2 * i], w[0][j + 2 * i + 1], w[1][j + 2 * i + 1], wh[i], wl[i]);
        add_products<T>(acc[m], wh, wl, s);
    };
    if constexpr (VEC && MB * sizeof(T) == 8) {
        // one piece; its registers take the next one's weights, 16 ranks after 16 (two pieces do not fit: 61 rows x 4096, 40 fp16
        // adapters of rank 64, both products 25.3 us, so 23.7)
        float v[8];
        T w[MB][2][8];
        if (k0 < k_end) {
            load_x(k0, v);
#pragma unroll
            for (int m = 0; m < MB; m++) load_a(k0, m, w[m]);
        }
#pragma unroll 1
        for (; k0 < k_end; k0 += step) {
            uint4 s[2][2];
            split_x(v, 0, s[0]), split_x(v, 4, s[1]);
            load_x(k0 + step, v);
#pragma unroll
            for (int m = 0; m < MB; m++) {
                multiply(m, w[m], 0, s[0]), multiply(m, w[m], 4, s[1]);
                load_a(k0 + step, m, w[m]);
            }
        }
    } else {
        // pieces on their way while one is multiplied, as the registers allow
        struct Piece {
            float v[8];
            T w[MB][2][8];
        };
        auto load = [&](int64_t k0, Piece& c) {
            load_x(k0, c.v);
#pragma unroll
            for (int m = 0; m < MB; m++) load_a(k0, m, c.w[m]);
        };
        constexpr int kDepth = VEC && MB * sizeof(T) < 8 ? DEPTH : 1;
        Piece c[kDepth];
#pragma unroll
        for (int d = 0; d + 1 < kDepth; d++)
            if (k0 + d * step < k_end) load(k0 + d * step, c[d]);
        while (k0 < k_end) {
#pragma unroll
            for (int d = 0; d < kDepth; d++) {
                if (k0 >= k_end) break;
                if (k0 + (kDepth - 1) * step < k_end) load(k0 + (kDepth - 1) * step, c[(d + kDepth - 1) % kDepth]);
#pragma unroll
                for (int j = 0; j < 8; j += 4) {
                    uint4 s[2];
                    split_x(c[d].v, j, s);
#pragma unroll
                    for (int m = 0; m < MB; m++) multiply(m, c[d].w[m], j, s);
                }
                k0 += step;
            }
        }
    }
}

// y += B t, or without `onto` y = B t, by one warp: 16 columns of NB times eight rows at a time, the next kAcross further; the next
// ones' first ranks of B are on their way meanwhile, and y is added to where it is (read and written back, its latency in each step:
// lora_add, 2048 rows x 4096 x 4096, 4 adapters of rank 32, 5.5 us more).  t is in shared memory, as the MMAs want it: two ranks of a
// row in 16 bytes, {hi, hi, lo, lo}, those that a lane reads in turn 64 bytes apart, rows `pitch` apart.
// QUADS: fours of ranks that a lane takes of a piece of 16 ranks (1, for at most 16) or 32 (2); PIECES of these at a time.
__host__ __device__ constexpr int expand_pitch(int ranks) { return ranks * 8 / 128 * 128 + 64 + (ranks * 8 % 128 > 64 ? 128 : 0); }  // bytes
template <typename T, int QUADS, int PIECES, int NB, int kAcross, bool VEC>
struct Columns {
    static constexpr int NV = 4 * QUADS, kPiece = 4 * NV, kChunk = kPiece * PIECES;  // values of a lane, ranks of a piece, ranks at a time
    struct Next {
        T w[PIECES][2][NV];
    };
    const T* b;          // of the lane's first values of column 0
    float* y;
    int64_t ldy;
    int y_row[NB][2];    // of row nb * 8 + 2t + i; where there is none, another's
    int n, N;            // the lane's columns: n and n + 1
    int rank, rows, live;  // rows from this warp's first on, blocks of eight that have any
    bool onto;
    Next c[2];

    // where pair i of a row's ranks stands in it
    static __device__ __forceinline__ int place(int i) {
        constexpr int kPairs = kPiece / 2, kOf = NV / 2;  // pair (NV / 2) t + j of a piece: at 4 j + t
        const int in = i % kPairs;
        return i / kPairs * kPairs + in % kOf * 4 + in / kOf;
    }
    // rows of the tile from `row0` of its place on, columns from n0 on
    __device__ __forceinline__ void begin(const LoraArgs& p, int4 tile, int tile_rows, int row0, int64_t n0, bool add) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        y = p.y, ldy = p.ldy, n = (int)n0 + 2 * g, N = (int)p.N, rank = p.rank, rows = tile_rows - row0, live = (rows + 7) / 8, onto = add;
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int row = nb * 8 + 2 * t + i;
                y_row[nb][i] = __ldcg(p.order + tile.y + (row < rows ? row0 + row : 0));
            }
        b = static_cast<const T*>(p.b) + (int64_t)tile.x * p.N * p.rank + NV * t;
    }
    // VEC: no branch and no predicate stands between these loads and what comes behind them, or the next piece would be waited for where it
    // is asked for.  So columns and ranks that do not exist read others': nothing of the former is stored, the latter are zeros in finish().
    __device__ __forceinline__ void load_b(int ahead, int r0, T (&w)[PIECES][2][NV]) {
        const int t = threadIdx.x & 3;
#pragma unroll
        for (int q = 0; q < PIECES; q++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int r = r0 + q * kPiece;
                const int m = n + ahead * kAcross + h;
                if constexpr (VEC)
                    load_values<NV, VEC>(b + ((int64_t)min(m, N - 1) * rank + (r + NV * t < rank ? r : -NV * t)), 1, w[q][h]);
                else
                    load_values<NV, VEC>(b + ((int64_t)m * rank + r), m < N ? rank - r - NV * t : 0, w[q][h]);
            }
    }
    __device__ __forceinline__ void finish(Next& c, const uint4* ts, int pitch) {
        float acc[NB][4] = {};
        const int lane = threadIdx.x & 31;
#pragma unroll 1
        for (int r0 = 0; r0 < rank; r0 += kChunk) {
            if (r0 > 0) load_b(0, r0, c.w);  // (more ranks than are held)
            const uint4* mine = ts + (lane >> 2) * pitch + r0 / 2 + (lane & 3);
#pragma unroll
            for (int q = 0; q < PIECES; q++) {
                if (VEC && r0 + q * kPiece + NV * (lane & 3) >= rank) {
#pragma unroll
                    for (int v = 0; v < NV; v++) c.w[q][0][v] = T(0.0f), c.w[q][1][v] = T(0.0f);
                }
#pragma unroll
                for (int j = 0; j < NV / 2; j += 2) {
                    uint32_t wh[2][4], wl[2][4];
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        operand(c.w[q][0][2 * (j + i)], c.w[q][1][2 * (j + i)], c.w[q][0][2 * (j + i) + 1], c.w[q][1][2 * (j + i) + 1], wh[i], wl[i]);
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) {
                        if (nb >= live) break;
                        const uint4* at = mine + nb * 8 * pitch + q * (kPiece / 2) + 4 * j;
                        const uint4 u[2] = {at[0], at[4]};
                        add_products<T>(acc[nb], wh, wl, u);
                    }
                }
            }
        }
        // acc[nb][i]: column n + i / 2 of row nb * 8 + 2t + i % 2
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (nb * 8 + 2 * (lane & 3) + i >= rows) continue;
                float* y = this->y + (y_row[nb][i] * ldy + n);
                if (onto) {
                    if (VEC && n < N) add_to(y, acc[nb][i], acc[nb][i + 2]);
                    if (!VEC && n < N) atomicAdd(y, acc[nb][i]);
                    if (!VEC && n + 1 < N) atomicAdd(y + 1, acc[nb][i + 2]);
                } else {
                    if (VEC && n < N) *reinterpret_cast<float2*>(y) = make_float2(acc[nb][i], acc[nb][i + 2]);
                    if (!VEC && n < N) y[0] = acc[nb][i];
                    if (!VEC && n + 1 < N) y[1] = acc[nb][i + 2];
                }
            }
        n += kAcross;
    }
    // `times` of them; the first one's B has been asked for into c[0]
    __device__ __forceinline__ void run(int64_t times, const uint4* ts, int pitch) {
#pragma unroll 1
        for (int64_t k = 0; k < times; k += 2) {
            if (k + 1 < times) load_b(1, 0, c[1].w);
            finish(c[0], ts, pitch);
            if (k + 1 >= times) break;
            if (k + 2 < times) load_b(1, 0, c[0].w);
            finish(c[1], ts, pitch);
        }
    }
};
// rows without an adapter, from the first-th on
__device__ __forceinline__ void zero_rows(const LoraArgs& p, int64_t first, int64_t step, int64_t n_begin, int64_t n_end) {
    for (int64_t i = __ldcg(p.offsets + p.n) + first; i < p.rows; i += step) {
        float* y = p.y + (int64_t)__ldcg(p.order + i) * p.ldy;
        for (int64_t n = n_begin + threadIdx.x; n < n_end; n += kThreads) y[n] = 0.0f;
    }
}

// ---- few rows and up to 64 ranks: both products in one launch ---------------------------------------------------------------------------
// A cluster per tile of eight rows: its CTAs divide K (and their warps that again), their sums meet in every one of them, and then they
// divide the columns.  With `early` the launch in front computes y alone: all else is complete, and the first product does not wait
// for it (12 rows x 6528 x 3057, 8 bf16 adapters of rank 24, with plan and FC 24.6 us, so 19.9): x and A in wide loads behind a fence, or value
// by value past L1 (through it, behind a fence, 133 rows x 1001 x 2999, 3 fp32 adapters of rank 12, 22.0 us, waiting 21.4, so 20.5).  CTAs
// behind those of the tiles quantize x for the decode FC (quant_pre.cuh), which has to be done in front of it anyway.
// Registers: two CTAs on an SM, and up to 32 ranks one beside a CTA of the prefill GEMM (16 rows x 4096 x 4096, 4 bf16 adapters of rank 16, with
// the FC: 118 registers 19.9 us, 96 18.5; 64 rows, 16 of rank 32, 128 registers 27.3, 112, and two pieces on their way instead of three, 26.9).
template <typename T, int MB, bool VEC_A, bool VEC_B>
__global__ void __maxnreg__(MB == 1 ? 96 : MB == 2 && (sizeof(T) == 2 || !VEC_A) ? 112 : 128)
    lora_few_kernel(const __grid_constant__ LoraArgs p, const __grid_constant__ QuantPre q, const bool onto, const bool early) {
    constexpr int kRanks = MB * 16, QUADS = MB == 1 ? 1 : 2, PIECES = MB == 4 && sizeof(T) < 4 ? 2 : 1, kAcross = kWarps * 16;
    using C = Columns<T, QUADS, PIECES, 1, kAcross, VEC_B>;
    constexpr int kPitch = expand_pitch((kRanks + C::kChunk - 1) / C::kChunk * C::kChunk) / 16;
    __shared__ float sums[8 * kRanks];                 // this CTA's [row][rank]
    __shared__ float by_warp[kWarps * 8 * kRanks];
    __shared__ uint4 ts[8 * kPitch];
    cg::cluster_group cluster = cg::this_cluster();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int slices = (int)gridDim.x, here = (int)blockIdx.x;
    auto others_done = [&] {
        pdl_wait_prior_grid();
        pdl_launch_dependents();
    };
    if (VEC_A && early) pdl_reads_early();  // (value by value x and A come past L1)
    if (!early) others_done();
    if ((int)blockIdx.y >= q.first_block) {
        quant_pre_block(q, ((int64_t)(blockIdx.y - q.first_block) * slices + here) * kWarps + warp);
        return;
    }
    const int64_t blocks = (p.N + kAcross - 1) / kAcross;
    const int64_t first = blocks * here / slices, times = blocks * (here + 1) / slices - first;
    const int4 tile = __ldcg(p.tiles + blockIdx.y);  // (beyond the count: nothing that is used)
    if ((int)blockIdx.y < __ldcg(p.tile_count)) {
        const int64_t k_begin = here * p.slice_k, k_end = min(p.K, k_begin + p.slice_k);
        const bool live = g < tile.z;
        const float* x = p.x + (live ? (int64_t)__ldcg(p.order + tile.y + g) * p.ldx : 0);
        float acc[MB][4] = {};
        shrink_rows<T, MB, VEC_A, !VEC_A, MB == 2 ? 2 : 3>(x, live, static_cast<const T*>(p.a) + (int64_t)tile.x * p.rank * p.K, p.rank, p.K,
                                                           k_begin + warp * 32, k_end, kWarps * 32, acc);
        float* mine = by_warp + warp * 8 * kRanks;
#pragma unroll
        for (int m = 0; m < MB; m++)
#pragma unroll
            for (int i = 0; i < 4; i++) mine[(2 * t + i % 2) * kRanks + m * 16 + 8 * (i / 2) + g] = acc[m][i];
        __syncthreads();
        for (int i = threadIdx.x; i < 8 * kRanks; i += kThreads) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) sum += by_warp[w * 8 * kRanks + i];
            sums[i] = sum;
        }
        if (early) others_done();
        C cols;
        cols.begin(p, tile, tile.z, 0, (first * kWarps + warp) * 16, onto);
        if (times > 0) cols.load_b(0, 0, cols.c[0].w);
        cluster.sync();
        const float scale = p.scales ? p.scales[tile.x] : 1.0f;
        for (int i = threadIdx.x; i < 8 * kRanks / 2; i += kThreads) {
            const int row = i / (kRanks / 2), r = i % (kRanks / 2) * 2;
            float v[2] = {0.0f, 0.0f};
            for (int s = 0; s < slices; s++) {
                const float2 o = *reinterpret_cast<const float2*>(cluster.map_shared_rank(sums, s) + row * kRanks + r);
                v[0] += o.x, v[1] += o.y;
            }
            uint4 u;
            split(v[0] * scale, u.x, u.z), split(v[1] * scale, u.y, u.w);
            ts[row * kPitch + C::place(r / 2)] = u;
        }
        __syncthreads();
        cols.run(times, ts, kPitch);
        cluster.sync();  // nobody leaves while its sums are being read
    } else if (early) {
        others_done();
    }
    if (!onto) zero_rows(p, blockIdx.y, q.first_block, first * kAcross, min(p.N, (first + times) * kAcross));
}

// ---- more rows, or more ranks: two launches ---------------------------------------------------------------------------------------------
// TILE rows: 64, eight warps with eight rows each, or 8, eight warps that divide the slice's K.  MB: 16-rank blocks in use.
template <typename T, int TILE, int MB, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) lora_shrink_kernel(const __grid_constant__ LoraArgs p) {
    constexpr bool kByK = TILE == 8;
    constexpr int kRanks = MB * 16;
    __shared__ float sums[TILE * kRanks];                     // this CTA's [row][rank]
    __shared__ float by_warp[kByK ? kWarps * TILE * kRanks : 1];
    cg::cluster_group cluster = cg::this_cluster();
    pdl_wait_prior_grid();
    __threadfence();  // expand reads the plan before this launch has ended (see DependentLaunch)
    pdl_launch_dependents();
    const int slices = (int)cluster.num_blocks(), here = (int)cluster.block_rank(), at = (int)blockIdx.x / slices;  // (clusters lie along x)
    const int4 tile = __ldcg(p.tiles + at);  // (beyond the count: nothing that is used)
    if (at >= __ldcg(p.tile_count)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int row0 = kByK ? 0 : warp * 8;
    const int rank0 = blockIdx.z * kRankBlock;
    const int64_t k_begin = here * p.slice_k, k_end = min(p.K, k_begin + p.slice_k);
    const bool live = row0 + g < tile.z;
    const float* x = p.x + (live ? (int64_t)__ldcg(p.order + tile.y + row0 + g) * p.ldx : 0);
    float acc[MB][4] = {};
    if (row0 < tile.z)
        shrink_rows<T, MB, VEC, false, 3>(x, live, static_cast<const T*>(p.a) + ((int64_t)tile.x * p.rank + rank0) * p.K, p.rank - rank0, p.K,
                                k_begin + (kByK ? warp * 32 : 0), k_end, kByK ? kWarps * 32 : 32, acc);
    float* mine = kByK ? by_warp + warp * TILE * kRanks : sums + row0 * kRanks;
#pragma unroll
    for (int m = 0; m < MB; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) mine[(2 * t + i % 2) * kRanks + m * 16 + 8 * (i / 2) + g] = acc[m][i];
    if constexpr (kByK) {
        __syncthreads();
        for (int i = threadIdx.x; i < TILE * kRanks; i += kThreads) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) sum += by_warp[w * TILE * kRanks + i];
            sums[i] = sum;
        }
    }
    cluster.sync();
    const float scale = p.scales ? p.scales[tile.x] : 1.0f;
    for (int i = here * kThreads + threadIdx.x; i < tile.z * kRanks; i += slices * kThreads) {
        float sum = 0.0f;
        for (int s = 0; s < slices; s++) sum += cluster.map_shared_rank(sums, s)[i];
        const int row = i / kRanks, r = i % kRanks;
        if (rank0 + r < p.rank) p.t[(int64_t)(tile.y + row) * p.rank + rank0 + r] = sum * scale;
    }
    cluster.sync();  // nobody leaves while its sums are being read
}

// The work is pieces of 32 rows of a tile and 64 columns, or of its eight rows and 128, the columns of a tile one behind another; a CTA
// takes a contiguous share of what the plan has.  (Both launches of lora_add with 2, 3 and 4 CTAs an SM: tiles of 64 rows, 2048 rows x
// 4096 x 4096, 4 bf16 adapters of rank 32, 39.0, 38.6 and 38.7 us; of eight, 61 rows x 4096 x 11008, 40 fp16 ones of rank 64, 23.4, 22.8 and
// 24.3.  Four times eight rows a warp instead of two: the same.  With fp32 weights of more than 16 ranks 2 hold the tiles of 64 rows without
// spilling: 1024 rows x 4096 x 4096, 8 adapters of rank 128, with 3 and 2 90.3 and 86.3 us.)
__host__ __device__ constexpr int expand_rows(int tile) { return tile < 32 ? tile : 32; }
__host__ __device__ constexpr int expand_columns(int tile) { return tile < 32 ? 128 : 64; }
// CTAs an SM; each: bytes of a weight
__host__ __device__ constexpr int expand_ctas(int each, int tile, int quads) { return each == 4 && quads == 2 && tile == 64 ? 2 : 3; }
template <typename T, int TILE, int QUADS, int PIECES, bool VEC>
__global__ void __launch_bounds__(kThreads, expand_ctas(sizeof(T), TILE, QUADS)) lora_expand_kernel(const __grid_constant__ LoraArgs p, const bool onto) {
    constexpr int kRows = expand_rows(TILE), kParts = TILE / kRows, NB = kRows > 8 ? 2 : 1, kAcross = expand_columns(TILE);
    using C = Columns<T, QUADS, PIECES, NB, kAcross, VEC>;
    extern __shared__ uint4 ts[];  // [kRows][pitch]
    const int pairs = (p.rank + C::kChunk - 1) / C::kChunk * C::kChunk / 2, pitch = expand_pitch(2 * pairs) / 16;
    // The launches in front, from shrink on, write t and y.  All else was complete when shrink had waited, and this launch begins only
    // after that: the plan and, VEC, B need not wait.  (Value by value, behind the fence: lora_add, 2048 rows x 4095 x 4095, 4 bf16 adapters of
    // rank 24, 62.0 us, so 58.4.)
    bool waited = false;
    auto others_done = [&] {
        if (!waited) {
            pdl_wait_prior_grid();
            pdl_launch_dependents();
        }
        waited = true;
    };
    if constexpr (VEC) pdl_reads_early();
    else others_done();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t blocks = (p.N + kAcross - 1) / kAcross, total = (int64_t)__ldcg(p.tile_count) * kParts * blocks;
    int64_t at = total * blockIdx.x / gridDim.x;
    const int64_t end = total * (blockIdx.x + 1) / gridDim.x;
    while (at < end) {
        const int64_t part = at / blocks;  // of a tile
        const int64_t first = at - part * blocks, last = min(blocks, first + end - at);
        at += last - first;
        int4 tile = __ldcg(p.tiles + part / kParts);
        tile.y += kRows * (int)(part % kParts), tile.z -= kRows * (int)(part % kParts);  // this piece's rows of it
        if (tile.z <= 0) continue;
        const int rows = min(tile.z, kRows), row0 = warp * 16 / kAcross * 16;  // (this warp's first row)
        C cols;
        cols.begin(p, tile, rows, row0, first * kAcross + warp * 16 % kAcross, onto);
        cols.load_b(0, 0, cols.c[0].w);
        others_done();
        __syncthreads();  // (nobody reads the piece in front any more)
        for (int row = warp; row < kRows; row += kWarps)
            for (int i = lane; i < pairs; i += 32) {
                float v[2] = {0.0f, 0.0f};
                if (row < rows) {
                    const float* from = p.t + (int64_t)(tile.y + row) * p.rank + 2 * i;
                    if (2 * i < p.rank) v[0] = __ldcg(from);
                    if (2 * i + 1 < p.rank) v[1] = __ldcg(from + 1);
                }
                uint4 u;
                split(v[0], u.x, u.z), split(v[1], u.y, u.w);
                ts[row * pitch + C::place(i)] = u;
            }
        __syncthreads();
        cols.run(last - first, ts + row0 * pitch, pitch);
    }
    others_done();
    if (!onto) zero_rows(p, blockIdx.x, gridDim.x, 0, p.N);
}

enum Step { kShrink, kExpand, kExpandOnto };
struct LoraPlan {
    int which, slices;
    int64_t slice_k, tiles;  // tiles that are likely in use
};
// Tiles of 64 rows from 256 rows on.  K in slices until the tiles that are likely in use fill the SMs twice, none below 256 k.
LoraPlan lora_plan(int64_t rows, int64_t K, int64_t rank, int64_t n, int sms) {
    LoraPlan l;
    l.which = rows >= 256 ? kTiles64 : kTiles8;
    const int64_t filled = rows / tile_rows(l.which), used = (n < rows ? n : rows) * 2 / 3;
    l.tiles = filled > used ? filled : used > 1 ? used : 1;
    const int64_t blocks = l.tiles * ((rank + kRankBlock - 1) / kRankBlock);
    int64_t slices = (2 * sms + blocks - 1) / blocks;
    const int64_t most = (K + 255) / 256 < kMostSlices ? (K + 255) / 256 : kMostSlices;
    if (slices > most) slices = most;
    l.slice_k = ((K + slices - 1) / slices + 31) / 32 * 32;
    l.slices = (int)((K + l.slice_k - 1) / l.slice_k);
    return l;
}

bool shrink_vec(const LoraCall& c) {
    return c.K % 8 == 0 && c.ldx % 4 == 0 && ((reinterpret_cast<uintptr_t>(c.x) | reinterpret_cast<uintptr_t>(c.a)) & 15) == 0;
}
bool expand_vec(const LoraCall& c, int values) {
    return c.rank % values == 0 && (reinterpret_cast<uintptr_t>(c.b) & 15) == 0 && c.N % 2 == 0 && c.ldy % 2 == 0 &&
           (reinterpret_cast<uintptr_t>(c.y) & 7) == 0;
}
// clusters of `ctas` along x
struct ClusterLaunch : DependentLaunch {
    cudaLaunchAttribute attrs[2];
    ClusterLaunch(dim3 grid, int ctas, cudaStream_t s) : DependentLaunch(grid, kThreads, s), attrs{attr, {}} {
        attrs[1].id = cudaLaunchAttributeClusterDimension;
        attrs[1].val.clusterDim.x = (unsigned)ctas, attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
        cfg.attrs = attrs, cfg.numAttrs = 2;
    }
};
template <typename T, int MB>
int launch_few(const LoraCall& c, const LoraArgs& p, const QuantPre& q, bool onto, bool early, dim3 grid, cudaStream_t s) {
    ClusterLaunch l(grid, (int)grid.x, s);
    const bool vec_b = expand_vec(c, MB == 1 ? 4 : 8);
    auto* fn = shrink_vec(c) ? vec_b ? lora_few_kernel<T, MB, true, true> : lora_few_kernel<T, MB, true, false>
                             : vec_b ? lora_few_kernel<T, MB, false, true> : lora_few_kernel<T, MB, false, false>;
    Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, fn, p, q, onto, early));
    return Q4FC_OK;
}
template <typename T, int TILE, int MB>
int launch_shrink(const LoraArgs& p, bool vec, dim3 grid, int slices, cudaStream_t s) {
    ClusterLaunch l(grid, slices, s);
    Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, vec ? lora_shrink_kernel<T, TILE, MB, true> : lora_shrink_kernel<T, TILE, MB, false>, p));
    return Q4FC_OK;
}
template <typename T, int TILE, int QUADS, int PIECES>
int launch_expand(const LoraCall& c, const LoraArgs& p, bool onto, int64_t tiles, cudaStream_t s) {
    const DeviceInfo* di = device_info();
    if (!di) return Q4FC_ECUDA;
    const bool vec = expand_vec(c, 4 * QUADS);
    constexpr int kChunk = 16 * QUADS * PIECES;
    const int64_t pieces = tiles * (TILE / expand_rows(TILE)) * ((c.N + expand_columns(TILE) - 1) / expand_columns(TILE));
    const int64_t most = expand_ctas(sizeof(T), TILE, QUADS) * di->sm_count;
    DependentLaunch l(dim3((unsigned)(pieces < most ? pieces : most)), kThreads, s);
    auto* fn = vec ? lora_expand_kernel<T, TILE, QUADS, PIECES, true> : lora_expand_kernel<T, TILE, QUADS, PIECES, false>;
    l.cfg.dynamicSmemBytes = expand_rows(TILE) * (size_t)expand_pitch((int)(c.rank + kChunk - 1) / kChunk * kChunk);
    // (what the highest rank needs, whatever this call's: a limit of its own would be another host thread's between that one's launch and its own)
    constexpr int kMost = expand_rows(TILE) * expand_pitch(kMostRanks);
    if constexpr (kMost > 48 * 1024) {
        static std::atomic<bool> attr_done[2][64] = {};  // set once per device; a second setter repeats the same call
        if (di->index >= 64 || !attr_done[vec][di->index]) {
            Q4FC_CUDA_OK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
            if (di->index < 64) attr_done[vec][di->index] = true;
        }
    }
    Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, fn, p, onto));
    return Q4FC_OK;
}
template <typename T, int TILE>
int launch_lora_tile(const LoraCall& c, const LoraArgs& p, const LoraPlan& l, Step step, int64_t tiles, cudaStream_t s) {
    if (step == kShrink) {
        const bool vec = shrink_vec(c);
        const dim3 grid((unsigned)(l.slices * tiles), 1, (unsigned)((c.rank + kRankBlock - 1) / kRankBlock));
        if (c.rank <= 16) return launch_shrink<T, TILE, 1>(p, vec, grid, l.slices, s);
        if (c.rank <= 32) return launch_shrink<T, TILE, 2>(p, vec, grid, l.slices, s);
        return launch_shrink<T, TILE, 4>(p, vec, grid, l.slices, s);
    }
    if (c.rank <= 16) return launch_expand<T, TILE, 1, 1>(c, p, step == kExpandOnto, tiles, s);
    if constexpr (sizeof(T) == 2)
        if (c.rank > 32) return launch_expand<T, TILE, 2, 2>(c, p, step == kExpandOnto, tiles, s);
    return launch_expand<T, TILE, 2, 1>(c, p, step == kExpandOnto, tiles, s);
}
template <typename T>
int launch_lora_type(const LoraCall& c, const LoraArgs& p, const LoraPlan& l, Step step, int64_t tiles, cudaStream_t s) {
    return l.which == kTiles8 ? launch_lora_tile<T, 8>(c, p, l, step, tiles, s) : launch_lora_tile<T, 64>(c, p, l, step, tiles, s);
}
int lora_args(const LoraCall& c, LoraPlan* l, LoraArgs* p, int64_t* tiles) {
    const DeviceInfo* di = device_info();
    if (!di) return Q4FC_ECUDA;
    *l = lora_plan(c.rows, c.K, c.rank, c.n, di->sm_count);
    *tiles = most_tiles(l->which, c.rows, c.n);
    *p = LoraArgs{c.x, c.a, c.b, c.scales, c.y, static_cast<float*>(c.scratch), c.plan.tiles[l->which], c.plan.counts + l->which, c.plan.order,
                  c.rows, c.K, c.ldx, c.N, c.ldy, l->slice_k, (int)c.rank, (int)c.n, c.plan.offsets};
    return Q4FC_OK;
}
int launch_lora(const LoraCall& c, Step step, cudaStream_t s) {
    LoraPlan l;
    LoraArgs p;
    int64_t tiles;
    if (int rc = lora_args(c, &l, &p, &tiles)) return rc;
    if (c.dtype == Q4FC_F32) return launch_lora_type<float>(c, p, l, step, tiles, s);
    if (c.dtype == Q4FC_F16) return launch_lora_type<__half>(c, p, l, step, tiles, s);
    return launch_lora_type<__nv_bfloat16>(c, p, l, step, tiles, s);
}
// Both products in one launch where each CTA of the second would have few of the columns anyway.  In one launch and in two, with the FC: 133
// rows x 1001 x 2999, fp32, rank 12, 20.3 and 21.8 us, 8 rows x 4096 x 4096, rank 16, 12.7 and 12.7; but 61 rows x 4096 x 11008, rank 64, 48.5
// and 43.0.
bool few(const LoraCall& c) {
    if (c.rows >= 256 || c.rank > kRankBlock) return false;
    const DeviceInfo* di = device_info();
    return di && lora_plan(c.rows, c.K, c.rank, c.n, di->sm_count).tiles * ((c.N + expand_columns(8) - 1) / expand_columns(8)) <= 4 * di->sm_count;
}
int launch_lora_few(const LoraCall& c, QuantPre q, bool onto, bool early, cudaStream_t s) {
    LoraPlan l;
    LoraArgs p;
    int64_t tiles;
    if (int rc = lora_args(c, &l, &p, &tiles)) return rc;
    q.first_block = (int)tiles;
    const int64_t warps = (int64_t)l.slices * kWarps, quant = (q.units() + warps - 1) / warps;
    const dim3 grid((unsigned)l.slices, (unsigned)(tiles + quant));
    auto with = [&](auto type) {
        using T = decltype(type);
        if (c.rank <= 16) return launch_few<T, 1>(c, p, q, onto, early, grid, s);
        if (c.rank <= 32) return launch_few<T, 2>(c, p, q, onto, early, grid, s);
        return launch_few<T, 4>(c, p, q, onto, early, grid, s);
    };
    if (c.dtype == Q4FC_F32) return with(float{});
    if (c.dtype == Q4FC_F16) return with(__half{});
    return with(__nv_bfloat16{});
}

}  // namespace

size_t lora_scratch_bytes(int64_t rows, int64_t rank) { return (size_t)(rows * rank) * 4; }

int launch_lora_add(const LoraCall& c, cudaStream_t s) {
    if (few(c)) return launch_lora_few(c, QuantPre{}, true, false, s);
    if (int rc = launch_lora(c, kShrink, s)) return rc;
    return launch_lora(c, kExpandOnto, s);
}

int launch_lora_first(const LoraCall& c, const QuantPre& q, cudaStream_t s) {
    if (few(c)) return launch_lora_few(c, q, false, false, s);
    if (int rc = launch_quant_x_pre(q.x, q.rows, q.K, q.ldx, q.G, q.want_isum, q.codes, q.sc, false, s)) return rc;
    if (int rc = launch_lora(c, kShrink, s)) return rc;
    return launch_lora(c, kExpand, s);
}

int launch_lora_before(const LoraCall& c, cudaStream_t s) { return few(c) ? Q4FC_OK : launch_lora(c, kShrink, s); }
int launch_lora_behind(const LoraCall& c, cudaStream_t s) {
    return few(c) ? launch_lora_few(c, QuantPre{}, true, true, s) : launch_lora(c, kExpandOnto, s);
}

}  // namespace q4fc
