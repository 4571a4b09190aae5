// Low-rank adapters beside a shared projection: y[m] += scale_i * B_i (A_i x[m]) for the adapter i of row m, the rows of a
// call in groups (groups.cuh).  No counterpart in the reference.  x is not quantized; A_i [rank][K] and B_i [N][rank] are
// fp32, fp16 or bf16 as the adapter was trained.
//
// Two launches, around whatever computes y:
//   shrink: t = A_i x, a CTA per tile of the plan's rows, slice of K and 64 ranks; slices are summed by expand, in order.
//   expand: y += scale_i * B_i t, a CTA per tile and 128 columns.
// Both on mma.sync.m16n8k8 (tf32 operands, fp32 sums), the adapter's rows on the 16-row side and the call's rows on the
// 8-column side.  A tf32 operand keeps 11 bits: fp16 and bf16 weights are exact in one, an fp32 number is two (its first 11
// bits and the rest, rounded), so that a product costs two MMAs, or three with fp32 weights, and is off by 2^-22.
// The order of k in an MMA is free as long as both operands have the same: a lane takes consecutive k of a row (8 of a piece
// of 32 in shrink, 4 of 16 in expand), so that fragments come straight from global memory in 16-byte loads.
#include <cuda_bf16.h>

#include <cfloat>

#include "groups.cuh"

namespace q4fc {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kRankBlock = 64;   // ranks of a CTA in shrink
constexpr int kColumns = 128;    // columns of a CTA in expand

// D(16x8) += A(16x8) * B(8x8)
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo: hi x's first 11 bits (cut off, which cannot overflow), lo the rest rounded to 11 bits
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
    hi = __float_as_uint(x) & 0xffffe000u;
    const float rest = fabsf(x) <= FLT_MAX ? x - __uint_as_float(hi) : 0.0f;  // (infinities and NaN are in hi)
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(rest));
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
        for (int i = 0; i < NV; i++) v[i] = i < valid ? p[i] : T(0.0f);
    }
}

struct LoraArgs {
    const float* x;
    const void *a, *b;
    const float* scales;   // of the adapters, or null
    float* y;
    float* part;           // [slice][row place][rank]
    const int4* tiles;
    const int *tile_count, *order;
    int64_t rows, K, ldx, N, ldy, slice_k;
    int rank, slices;
};

// TILE rows: 64, eight warps with eight rows each, or 8, eight warps that divide the slice's K.  MB: 16-rank blocks in use.
template <typename T, int TILE, int MB, bool VEC>
__global__ void __launch_bounds__(kThreads) lora_shrink_kernel(const __grid_constant__ LoraArgs p) {
    constexpr bool kByK = TILE == 8;
    __shared__ float sums[kByK ? kWarps * MB * 16 * 8 : 1];
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    if ((int)blockIdx.y >= __ldcg(p.tile_count)) return;
    const int4 tile = __ldcg(p.tiles + blockIdx.y);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int row0 = kByK ? 0 : warp * 8;
    if (!kByK && row0 >= tile.z) return;
    const int rank0 = blockIdx.z * kRankBlock;
    const int64_t k_begin = blockIdx.x * p.slice_k, k_end = min(p.K, k_begin + p.slice_k);
    const bool live = row0 + g < tile.z;
    const float* x = p.x + (live ? (int64_t)__ldcg(p.order + tile.y + row0 + g) * p.ldx : 0);
    const T* a = static_cast<const T*>(p.a) + ((int64_t)tile.x * p.rank + rank0) * p.K;
    float acc[MB][4] = {};
    for (int64_t k0 = k_begin + (kByK ? warp * 32 : 0); k0 < k_end; k0 += kByK ? kWarps * 32 : 32) {
        const int64_t k = k0 + 8 * t;
        float v[8];
        T w[MB][2][8];
        load_values<8, VEC>(x + k, live ? k_end - k : 0, v);
#pragma unroll
        for (int m = 0; m < MB; m++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int r = m * 16 + h * 8 + g;
                load_values<8, VEC>(a + (int64_t)r * p.K + k, rank0 + r < p.rank ? k_end - k : 0, w[m][h]);
            }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t hi0, lo0, hi1, lo1;
            split(v[2 * j], hi0, lo0), split(v[2 * j + 1], hi1, lo1);
#pragma unroll
            for (int m = 0; m < MB; m++) {
                const float f[4] = {number(w[m][0][2 * j]), number(w[m][1][2 * j]), number(w[m][0][2 * j + 1]), number(w[m][1][2 * j + 1])};
                uint32_t wh[4], wl[4];
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int i = 0; i < 4; i++) split(f[i], wh[i], wl[i]);
                    mma_tf32(acc[m], wl, hi0, hi1);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) wh[i] = __float_as_uint(f[i]);
                }
                mma_tf32(acc[m], wh, lo0, lo1);
                mma_tf32(acc[m], wh, hi0, hi1);
            }
        }
    }
    // acc[m][i]: rank m * 16 + 8 (i / 2) + g of row 2t + i % 2
    float* part = p.part + ((int64_t)blockIdx.x * p.rows + tile.y) * p.rank + rank0;
    if constexpr (kByK) {
#pragma unroll
        for (int m = 0; m < MB; m++)
#pragma unroll
            for (int i = 0; i < 4; i++) sums[((warp * 8 + 2 * t + i % 2) * MB + m) * 16 + 8 * (i / 2) + g] = acc[m][i];
        __syncthreads();
        for (int i = threadIdx.x; i < 8 * MB * 16; i += kThreads) {
            const int row = i / (MB * 16), r = i % (MB * 16);
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) sum += sums[w * 8 * MB * 16 + i];
            if (row < tile.z && rank0 + r < p.rank) part[(int64_t)row * p.rank + r] = sum;
        }
    } else {
#pragma unroll
        for (int m = 0; m < MB; m++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = row0 + 2 * t + i % 2, r = m * 16 + 8 * (i / 2) + g;
                if (row < tile.z && rank0 + r < p.rank) part[(int64_t)row * p.rank + r] = acc[m][i];
            }
    }
}

// VEC: 4 ranks of a row of B in one load, two columns of y in one
template <typename T, int TILE, bool VEC>
__global__ void __launch_bounds__(kThreads) lora_expand_kernel(const __grid_constant__ LoraArgs p) {
    extern __shared__ float ts[];  // t of the tile: [TILE][pitch], scaled
    const int ranks = (p.rank + 15) / 16 * 16, pitch = ranks + 8;  // (rows 8 words apart: a float2 a lane without conflicts)
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    if ((int)blockIdx.y >= __ldcg(p.tile_count)) return;
    const int4 tile = __ldcg(p.tiles + blockIdx.y);
    const float scale = p.scales ? p.scales[tile.x] : 1.0f;
    for (int i = threadIdx.x; i < TILE * ranks; i += kThreads) {
        const int row = i / ranks, r = i - row * ranks;
        float sum = 0.0f;
        if (row < tile.z && r < p.rank) {
            const float* src = p.part + ((int64_t)tile.y + row) * p.rank + r;
#pragma unroll 4
            for (int s = 0; s < p.slices; s++) sum += __ldcg(src + (int64_t)s * p.rows * p.rank);
        }
        ts[row * pitch + r] = sum * scale;
    }
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t n = (int64_t)blockIdx.x * kColumns + warp * 16 + 2 * g;  // this lane's columns: n and n + 1
    if (n - 2 * g >= p.N) return;
    const T* b = static_cast<const T*>(p.b) + ((int64_t)tile.x * p.N + n) * p.rank;
    constexpr int NB = TILE / 8;
    const int blocks = (tile.z + 7) / 8;
    float acc[NB][4] = {};
    for (int r0 = 0; r0 < p.rank; r0 += 16) {
        const int r = r0 + 4 * t;
        T w[2][4];
#pragma unroll
        for (int h = 0; h < 2; h++) load_values<4, VEC>(b + h * p.rank + r, n + h < p.N ? p.rank - r : 0, w[h]);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const float f[4] = {number(w[0][2 * j]), number(w[1][2 * j]), number(w[0][2 * j + 1]), number(w[1][2 * j + 1])};
            uint32_t wh[4], wl[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                if constexpr (sizeof(T) == 4) split(f[i], wh[i], wl[i]);
                else wh[i] = __float_as_uint(f[i]);
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                if (nb >= blocks) break;
                const float2 v = *reinterpret_cast<const float2*>(ts + (nb * 8 + g) * pitch + r + 2 * j);
                uint32_t hi0, lo0, hi1, lo1;
                split(v.x, hi0, lo0), split(v.y, hi1, lo1);
                if constexpr (sizeof(T) == 4) mma_tf32(acc[nb], wl, hi0, hi1);
                mma_tf32(acc[nb], wh, lo0, lo1);
                mma_tf32(acc[nb], wh, hi0, hi1);
            }
        }
    }
    // acc[nb][i]: column n + i / 2 of row nb * 8 + 2t + i % 2
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int row = nb * 8 + 2 * t + i;
            if (row >= tile.z) continue;
            float* y = p.y + (int64_t)__ldcg(p.order + tile.y + row) * p.ldy + n;
            if (VEC && n + 1 < p.N) {
                float2 v = __ldcg(reinterpret_cast<const float2*>(y));
                v.x += acc[nb][i], v.y += acc[nb][i + 2];
                *reinterpret_cast<float2*>(y) = v;
            } else {
                if (n < p.N) y[0] = __ldcg(y) + acc[nb][i];
                if (n + 1 < p.N) y[1] = __ldcg(y + 1) + acc[nb][i + 2];
            }
        }
}

struct LoraPlan {
    int which, slices;
    int64_t slice_k;
};
// Tiles of 64 rows from 256 rows on.  K in slices until the tiles that are likely in use fill the SMs twice, none below 256 k.
LoraPlan lora_plan(int64_t rows, int64_t K, int64_t rank, int64_t n, int sms) {
    LoraPlan l;
    l.which = rows >= 256 ? kTiles64 : kTiles8;
    const int64_t least = n < rows ? n : rows, tiles = rows / tile_rows(l.which) > least ? rows / tile_rows(l.which) : least;
    const int64_t blocks = tiles * ((rank + kRankBlock - 1) / kRankBlock);
    int64_t slices = (2 * sms + blocks - 1) / blocks;
    const int64_t most = (K + 255) / 256 < 16 ? (K + 255) / 256 : 16;
    if (slices > most) slices = most;
    l.slice_k = ((K + slices - 1) / slices + 31) / 32 * 32;
    l.slices = (int)((K + l.slice_k - 1) / l.slice_k);
    return l;
}

template <typename T, int TILE, int MB>
int launch_shrink(const LoraArgs& p, bool vec, dim3 grid, cudaStream_t s) {
    DependentLaunch l(grid, kThreads, s);
    Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, vec ? lora_shrink_kernel<T, TILE, MB, true> : lora_shrink_kernel<T, TILE, MB, false>, p));
    return Q4FC_OK;
}
template <typename T, int TILE>
int launch_lora_tile(const LoraCall& c, const LoraArgs& p, bool expand, int64_t tiles, cudaStream_t s) {
    if (!expand) {
        const bool vec = c.K % 8 == 0 && c.ldx % 4 == 0 && ((reinterpret_cast<uintptr_t>(c.x) | reinterpret_cast<uintptr_t>(c.a)) & 15) == 0;
        const dim3 grid((unsigned)p.slices, (unsigned)tiles, (unsigned)((c.rank + kRankBlock - 1) / kRankBlock));
        if (c.rank <= 16) return launch_shrink<T, TILE, 1>(p, vec, grid, s);
        if (c.rank <= 32) return launch_shrink<T, TILE, 2>(p, vec, grid, s);
        return launch_shrink<T, TILE, 4>(p, vec, grid, s);
    }
    const bool vec = c.rank % 4 == 0 && c.ldy % 2 == 0 && (reinterpret_cast<uintptr_t>(c.y) & 7) == 0 && (reinterpret_cast<uintptr_t>(c.b) & 15) == 0;
    DependentLaunch l(dim3((unsigned)((c.N + kColumns - 1) / kColumns), (unsigned)tiles), kThreads, s);
    auto* fn = vec ? lora_expand_kernel<T, TILE, true> : lora_expand_kernel<T, TILE, false>;
    l.cfg.dynamicSmemBytes = TILE * (size_t)((c.rank + 15) / 16 * 16 + 8) * 4;
    if (l.cfg.dynamicSmemBytes > 48 * 1024)
        Q4FC_CUDA_OK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)l.cfg.dynamicSmemBytes));
    Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, fn, p));
    return Q4FC_OK;
}
template <typename T>
int launch_lora_type(const LoraCall& c, const LoraArgs& p, int which, bool expand, int64_t tiles, cudaStream_t s) {
    return which == kTiles8 ? launch_lora_tile<T, 8>(c, p, expand, tiles, s) : launch_lora_tile<T, 64>(c, p, expand, tiles, s);
}
int launch_lora(const LoraCall& c, bool expand, cudaStream_t s) {
    const DeviceInfo* di = device_info();
    if (!di) return Q4FC_ECUDA;
    const LoraPlan l = lora_plan(c.rows, c.K, c.rank, c.n, di->sm_count);
    const int64_t tiles = most_tiles(l.which, c.rows, c.n);
    if (tiles > 65535) {
        set_error("lora: %lld rows exceed the grid limit", (long long)c.rows);
        return Q4FC_ELIMIT;
    }
    LoraArgs p = {c.x, c.a, c.b, c.scales, c.y, static_cast<float*>(c.scratch), c.plan.tiles[l.which], c.plan.counts + l.which, c.plan.order,
                  c.rows, c.K, c.ldx, c.N, c.ldy, l.slice_k, (int)c.rank, l.slices};
    if (c.dtype == Q4FC_F32) return launch_lora_type<float>(c, p, l.which, expand, tiles, s);
    if (c.dtype == Q4FC_F16) return launch_lora_type<__half>(c, p, l.which, expand, tiles, s);
    return launch_lora_type<__nv_bfloat16>(c, p, l.which, expand, tiles, s);
}

}  // namespace

// (slices do not depend on the card: at most 16)
size_t lora_scratch_bytes(int64_t rows, int64_t rank) { return (size_t)(rows * rank) * 16 * 4; }
int launch_lora_shrink(const LoraCall& c, cudaStream_t s) { return launch_lora(c, false, s); }
int launch_lora_expand(const LoraCall& c, cudaStream_t s) { return launch_lora(c, true, s); }

}  // namespace q4fc
