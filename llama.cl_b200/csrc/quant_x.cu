// Stand-alone Q8 activation quantizer.
//
// Replaces FC_dynamic_quantize_x (ops/op_fc.hpp:221-272) with get_amax and
// quant_row_q8_0 (ops/utils.hpp:177-220): per row and K group
//   amax = max|x|, d = amax/127, id = 1/d (0 when d == 0),
//   scales = d * scale, codes = sat_s8(round(x * id)), gsums = sum of raw x.
// Rounding follows the reference exactly: the first floor(len/8)*8 elements
// of a group round half to even (its 8-wide AVX2 body), the remaining
// len % 8 elements round half away from zero (its scalar tail); padding codes
// are 0.  The group sum is accumulated sequentially in k order so that it is
// bit-equal to the reference's loop (ops/op_fc.hpp:262-268).
//
// One warp owns 128 consecutive k of one row: a 512-byte coalesced read, four
// values per lane.  The absolute maximum is a segmented butterfly over the
// G/4 lanes of a group.  The raw values are parked in shared memory so that
// one lane per group can walk them in order for the sequential sum; many
// resident warps hide that serial chain.  The decode FC kernel has its own
// fused copy of this arithmetic (tree-ordered sums), the prefill path its own
// kernel below; this one serves callers that want the quantized activations
// themselves and the per-channel int8 FC on mma.sync (q8c.cu).
#include <type_traits>

#include "groups.cuh"
#include "quant_pre.cuh"

namespace q4fc {
namespace {

constexpr int kQxWarps = 8;

template <int G>
__global__ void __launch_bounds__(kQxWarps * 32) quant_x_kernel(const float* __restrict__ x, int64_t rows, int64_t K,
                                                                int64_t ldx, int64_t Kg, float scale, int vec_ok,
                                                                int8_t* __restrict__ codes, float* __restrict__ scales,
                                                                float* __restrict__ gsums) {
    constexpr int SEG = G / 4;     // lanes per group
    constexpr int GPC = 128 / G;   // groups per 128-k chunk
    constexpr int PADG = G + 1;    // padded group pitch in shared memory
    __shared__ float raw[kQxWarps][GPC * PADG + 3];

    pdl_wait_prior_grid();
    pdl_launch_dependents();  // (an FC launched for it starts beside this kernel and waits for its results)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t chunks = (Kg * G + 127) / 128;
    const int64_t unit = (int64_t)blockIdx.x * kQxWarps + warp;
    if (unit >= rows * chunks) return;
    const int64_t row = unit / chunks;
    const int64_t c = unit % chunks;
    const int64_t k = c * 128 + lane * 4;
    const float* src = x + row * ldx + k;

    float v[4];
    if (vec_ok && k + 4 <= K) {
        float4 a = ld_after_wait(reinterpret_cast<const float4*>(src));
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = (k + j < K) ? ld_after_wait(src + j) : 0.0f;
    }

    const int g_l = lane / SEG;              // group inside the chunk
    const int64_t kb = c * GPC + g_l;        // group index in the row
    const bool group_exists = kb < Kg;
    const int len = group_exists ? (int)min((int64_t)G, K - kb * G) : 0;
    const int body = (len / 8) * 8;
    const int e0 = (lane % SEG) * 4;         // element index of v[0] inside the group

    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (e0 + j < len) amax = fmaxf(amax, fabsf(v[j]));
#pragma unroll
    for (int off = SEG / 2; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off, SEG));

    const float d = div_const_rn(amax, 127.0f, 1.0f / 127.0f);
    const float id = inv_or_zero(d);

    uint32_t packed = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int e = e0 + j;
        int q = 0;
        if (e < len) {
            const float t = __fmul_rn(v[j], id);
            if (e < body) {
                q = sat8(__float2int_rn(t));  // nearest even, as _mm256_round_ps + packs
            } else {
                q = sat8(round_half_away(t));  // std::round
            }
        }
        packed |= (uint32_t)(q & 0xFF) << (8 * j);
    }
    if (group_exists) {
        *reinterpret_cast<uint32_t*>(codes + row * (Kg * G) + k) = packed;
        if (lane % SEG == 0) scales[row * Kg + kb] = __fmul_rn(d, scale);
    }

    if (gsums != nullptr) {
        float* mine = raw[warp];
#pragma unroll
        for (int j = 0; j < 4; j++) mine[g_l * PADG + e0 + j] = v[j];
        __syncwarp();
        if (lane < GPC) {
            const int64_t kb2 = c * GPC + lane;
            if (kb2 < Kg) {
                const int len2 = (int)min((int64_t)G, K - kb2 * G);
                float s = 0.0f;
                for (int i = 0; i < len2; i++) s = __fadd_rn(s, mine[lane * PADG + i]);
                gsums[row * Kg + kb2] = s;
            }
        }
    }
}

// 128 k of a row, by one warp, as the FC kernels read them: lane l holds v[0..3] = x[k .. k + 3], k = 4 l behind the first one; 0
// beyond K, which is `left` behind it.  Codes and scales as in quant_x_kernel, group sums tree-ordered.  isum: instead of the sum, the
// bits of the integer 8 * sum of codes.
struct QuantizedUnit {
    uint32_t w[2];  // the lane's codes: four bytes, or four fp16 (see launch_quant_x_tile)
    float scale, sum;
};
template <int G, bool F16>
__device__ __forceinline__ QuantizedUnit quantize_unit(const float (&v)[4], int lane, int left, bool isum) {
    constexpr int SEG = G / 4;    // lanes per group
    const int len = min(G, max(0, left - lane / SEG * G));  // of this lane's group
    const int body = len & ~7;
    const int e0 = (lane % SEG) * 4;
    float amax = fmaxf(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))), 0.0f);  // (0 of missing values alone)
    float sum = (v[0] + v[1]) + (v[2] + v[3]);
#pragma unroll
    for (int off = SEG / 2; off > 0; off >>= 1) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        sum += __shfl_xor_sync(0xffffffffu, sum, off);
    }
    const float d = div_const_rn(amax, 127.0f, 1.0f / 127.0f);
    const float id = inv_or_zero(d);
    uint32_t w[2] = {};  // F16: four codes, as two lanes hold eight k: the even one takes k = 0,2,4,6
    // Ordinary groups, whole: |v x id| < 128, and t + 1.5 x 2^23 rounds t to the nearest integer, half to even, and has it in its low bits.
    // (Missing values: fmaxf does not see them, the sum does.)
    const bool ordinary = (amax == 0.0f || (amax >= 0x1p-100f && amax <= 0x1p100f)) && sum == sum;
    if (left >= 128 && __all_sync(0xffffffffu, ordinary)) {
        float t[4];
#pragma unroll
        for (int j = 0; j < 4; j++) t[j] = __fadd_rn(__fmul_rn(v[j], id), 12582912.0f);
        const uint32_t lo = __byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040), hi = __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040);
        w[0] = __byte_perm(lo, hi, 0x5410);
        if constexpr (F16) {
            const float up = (lane & 1) ? 16.0f : 256.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) t[j] = __fmul_rn(__fadd_rn(t[j], -12582912.0f), up);
            const __half2 even2 = __floats2half2_rn(t[0], t[2]), odd2 = __floats2half2_rn(t[1], t[3]);
            const uint32_t even = *reinterpret_cast<const uint32_t*>(&even2), odd = *reinterpret_cast<const uint32_t*>(&odd2);
            const uint32_t other = __shfl_xor_sync(0xffffffffu, (lane & 1) ? even : odd, 1);
            w[0] = (lane & 1) ? other : even, w[1] = (lane & 1) ? odd : other;
        } else if (isum) {
            int s = __dp4a((int)w[0], 0x01010101, 0);
#pragma unroll
            for (int off = SEG / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
            sum = __int_as_float(8 * s);
        }
    } else {
        int q[4] = {};
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (e0 + j < len) {
                const float t = __fmul_rn(v[j], id);
                q[j] = sat8(e0 + j < body ? __float2int_rn(t) : round_half_away(t));
            }
        if (isum) {
            int s = q[0] + q[1] + q[2] + q[3];
#pragma unroll
            for (int off = SEG / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
            sum = __int_as_float(8 * s);
        }
        w[0] = (q[0] & 0xFF) | (q[1] & 0xFF) << 8 | (q[2] & 0xFF) << 16 | (uint32_t)(q[3] & 0xFF) << 24;
        if constexpr (F16) {
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; j++) h[j] = __half_as_ushort(__int2half_rn(q[j] * ((lane & 1) ? 16 : 256)));
            const uint32_t even = h[0] | h[2] << 16, odd = h[1] | h[3] << 16;
            const uint32_t other = __shfl_xor_sync(0xffffffffu, (lane & 1) ? even : odd, 1);
            w[0] = (lane & 1) ? other : even, w[1] = (lane & 1) ? odd : other;
        }
    }
    return {{w[0], w[1]}, F16 ? __fmul_rn(d, 64.0f) : d, sum};
}
// `codes`: the lane's place; `sc`: the row's place in the first of the 128 k's groups, `per` floats from there to its place in the next, the
// sum `sum_at` behind the scale.  groups: of the 128 k that are written.
template <int G, bool F16>
__device__ __forceinline__ void store_unit(const QuantizedUnit& q, int lane, int groups, bool sums, int8_t* codes, float* sc, int64_t per, int64_t sum_at) {
    constexpr int SEG = G / 4;
    if (lane / SEG >= groups) return;
    if constexpr (F16)
        *reinterpret_cast<uint2*>(codes) = make_uint2(q.w[0], q.w[1]);
    else
        *reinterpret_cast<uint32_t*>(codes) = q.w[0];
    if (lane % SEG == 0) {
        float* dst = sc + lane / SEG * per;
        dst[0] = q.scale;
        if (sums) dst[sum_at] = q.sum;
    }
}

// The lane's values of `CHUNKS` times 128 k from chunk c on, all asked for at once; 0 beyond K.
template <int CHUNKS>
__device__ __forceinline__ void load_chunks(const float* __restrict__ row, int64_t c, int lane, int64_t K, int vec_ok, float (&v)[CHUNKS][4]) {
#pragma unroll
    for (int i = 0; i < CHUNKS; i++) {
        const int64_t k = (c + i) * 128 + lane * 4;
        v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.0f;
        if (vec_ok && k + 4 <= K) {
            const float4 a = ld_after_wait(reinterpret_cast<const float4*>(row + k));
            v[i][0] = a.x, v[i][1] = a.y, v[i][2] = a.z, v[i][3] = a.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (k + j < K) v[i][j] = ld_after_wait(row + k + j);
        }
    }
}
// Chunks of a warp: many rows are quantized four at a time, so that a warp starts, and finds its row, a quarter as often (2048 x 4096
// 20 -> 18 us); few rows one at a time, for the shortest way through.
constexpr int kManyChunks = 4;
constexpr int64_t kManyUnits = 16384;  // rows x chunks

// The prefill GEMM's quantizer: the codes and scales of quant_x_kernel, scales (and, `sums`, group sums, tree-ordered)
// in the layout in which the GEMM's tiles of 2^log2tile rows read them: [row tile][Kg][scale | sum][row in tile].
// The eight warps of a CTA take the same k of eight neighbouring rows, whose scales share a 32-byte sector.
template <int G, bool F16, int CHUNKS>
__global__ void __launch_bounds__(kQxWarps * 32) quant_x_tile_kernel(const float* __restrict__ x, int64_t rows, int64_t K,
                                                                     int64_t ldx, int64_t Kg, int vec_ok, int sums,
                                                                     int log2tile, int8_t* __restrict__ codes,
                                                                     float* __restrict__ sc) {
    pdl_wait_prior_grid();
    pdl_launch_dependents();      // the GEMM's weight copies run beside this launch
    const int lane = threadIdx.x & 31;
    const int64_t row_sets = (rows + kQxWarps - 1) / kQxWarps;
    const int64_t set = blockIdx.x / row_sets, c = set * CHUNKS;
    const int64_t row = (blockIdx.x - set * row_sets) * kQxWarps + (threadIdx.x >> 5);
    if (row >= rows) return;
    float v[CHUNKS][4];
    load_chunks<CHUNKS>(x + row * ldx, c, lane, K, vec_ok, v);
    const int64_t tile = (int64_t)1 << log2tile, per = tile << sums;
    float* dst = sc + ((row >> log2tile) * Kg + c * (128 / G)) * per + (row & (tile - 1));
    int8_t* to = codes + (row * (Kg * G) + c * 128 + lane * 4) * (F16 ? 2 : 1);
    const int left = (int)min((int64_t)CHUNKS * 128, K - c * 128);
#pragma unroll
    for (int i = 0; i < CHUNKS; i++)
        if (CHUNKS == 1 || 128 * i < left)
            store_unit<G, F16>(quantize_unit<G, F16>(v[i], lane, left - 128 * i, false), lane, (left - 128 * i + G - 1) / G, sums,
                               to + 128 * i * (F16 ? 2 : 1), dst + i * (128 / G) * per, per, tile);
}

// The quantizer of the experts' product: a row of x for each of its `per_row` (token, slot) pairs, or one; codes in the order of the
// plan (groups.cuh), scales by its tiles: for experts with few rows (tiles of 16) [tile][K group][two rows][scales, sums], else
// as quant_x_tile_kernel has them.  `gated`: the value is silu(x[k]) * x[K + k].  An output row without an expert is zeroed here.
template <int G, bool F16, int CHUNKS>
__global__ void __launch_bounds__(kQxWarps * 32) quant_x_group_kernel(const __grid_constant__ GroupQuant a) {
    pdl_wait_prior_grid();
    __threadfence();              // what is behind this launch reads the plan, too, before this launch has ended (see DependentLaunch)
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t x_rows = a.rows / a.per_row, row_sets = (x_rows + kQxWarps - 1) / kQxWarps;
    const int64_t set = blockIdx.x / row_sets, c = set * CHUNKS;
    const int64_t row = (blockIdx.x - set * row_sets) * kQxWarps + (threadIdx.x >> 5);
    if (row >= x_rows) return;
    float v[CHUNKS][4];
    load_chunks<CHUNKS>(a.x + row * a.ldx, c, lane, a.K, a.vec_ok, v);
    // lane s: where the codes and scales of slot s go; -1: nowhere
    const bool few = a.log2tile == 4;
    const int64_t chunks = (a.Kg * G + 127) / 128, size = (int64_t)1 << a.log2tile, per = few ? 32 : size << a.sums, sum_at = few ? 2 : size;
    int64_t code_at = -1, sc_at = 0;
    int group = a.n;
    if (lane < a.per_row) {
        const int64_t pair = row * a.per_row + lane;
        group = __ldcg(a.group_of + pair);
        const int64_t place = __ldcg(a.place_of + pair);
        if (group < a.n) {
            const int at = (int)place - __ldcg(a.offsets + group), in = at & ((1 << a.log2tile) - 1);
            const int64_t tile = __ldcg(a.tile0 + group) + (at >> a.log2tile);
            code_at = few ? (place * chunks + c) * 128 : (place * (a.Kg * G) + c * 128) * (F16 ? 2 : 1);
            sc_at = (tile * (few ? chunks * (128 / G) : a.Kg) + c * (128 / G)) * per + (few ? in / 2 * 4 + in % 2 : in);
        }
    }
    const uint32_t none = __ballot_sync(0xffffffffu, lane < a.per_row && group >= a.n);
    if (c == 0)
        for (uint32_t left = none; left; left &= left - 1)
            for (int64_t n = lane; n < a.N; n += 32) a.y[(row * a.per_row + __ffs(left) - 1) * a.ldy + n] = 0.0f;
    if (a.gated) {
        float up[CHUNKS][4];
        load_chunks<CHUNKS>(a.x + row * a.ldx + a.K, c, lane, a.K, a.vec_ok, up);
#pragma unroll
        for (int i = 0; i < CHUNKS; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) v[i][j] = __fmul_rn(up[i][j], __fdiv_rn(v[i][j], __fadd_rn(1.0f, expf(-v[i][j]))));
    }
    const int left = (int)min((int64_t)CHUNKS * 128, a.K - c * 128);
    QuantizedUnit q[CHUNKS];
#pragma unroll
    for (int i = 0; i < CHUNKS; i++)
        if (CHUNKS == 1 || 128 * i < left) q[i] = quantize_unit<G, F16>(v[i], lane, left - 128 * i, a.isum);
    // (what a lane of the FC kernel for few rows takes of 128 k -- eight of each 32 -- lies together; scales and sums of two rows do)
    const int mine = few ? (lane / 2 % 4) * 32 + (lane / 8) * 8 + (lane % 2) * 4 : lane * 4 * (F16 ? 2 : 1);
#pragma unroll 1
    for (int s = 0; s < a.per_row; s++) {
        const int64_t to = __shfl_sync(0xffffffffu, code_at, s), sc = __shfl_sync(0xffffffffu, sc_at, s);
        if (to < 0) continue;
#pragma unroll
        for (int i = 0; i < CHUNKS; i++)
            if (CHUNKS == 1 || 128 * i < left)
                store_unit<G, F16>(q[i], lane, few ? 128 / G : (left - 128 * i + G - 1) / G, few || a.sums,
                                   a.codes + to + mine + 128 * i * (F16 ? 2 : 1), a.sc + sc + i * (128 / G) * per, per, sum_at);
    }
}

// The quantizer in front of the decode FC: quant_pre.cuh.
template <int G>
__global__ void __launch_bounds__(128) quant_x_pre_kernel(const float* __restrict__ x, int rows, int64_t K,
                                                          int64_t ldx, int64_t Kg, int vec_ok, int want_isum,
                                                          int early_release, int8_t* __restrict__ codes,
                                                          float* __restrict__ sc, const float* __restrict__ up,
                                                          float* __restrict__ prod, int64_t ldp) {
    quant_pre_unit<G>(x, rows, K, ldx, Kg, vec_ok, want_isum, early_release, codes, sc, up, prod, ldp,
                      (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5));
}

// Several inputs in one launch (a batch of independent FCs has as many inputs to quantize, and each launch of its own
// would cost more than its work): the warps of the grid are dealt out to the inputs in order.
constexpr int kMaxQuantBatch = 16;
struct QuantBatch {
    const float* x[kMaxQuantBatch];
    int8_t* codes[kMaxQuantBatch];
    float* sc[kMaxQuantBatch];
    int64_t K[kMaxQuantBatch], ldx[kMaxQuantBatch];
    int rows[kMaxQuantBatch], vec_ok[kMaxQuantBatch];
    int unit0[kMaxQuantBatch + 1];  // first warp of input i; [n] = warps in all
    int n;
};
template <int G>
__global__ void __launch_bounds__(128) quant_x_pre_batch_kernel(const __grid_constant__ QuantBatch b, int want_isum,
                                                                int early_release) {
    const int unit = (int)blockIdx.x * 4 + (threadIdx.x >> 5);
    int i = 0;
    while (i + 1 < b.n && unit >= b.unit0[i + 1]) i++;
    const int64_t Kg = (b.K[i] + G - 1) / G;
    if (unit >= b.unit0[b.n]) {
        if (early_release) pdl_launch_dependents();
        return;
    }
    quant_pre_unit<G>(b.x[i], b.rows[i], b.K[i], b.ldx[i], Kg, b.vec_ok[i], want_isum, early_release, b.codes[i], b.sc[i],
                      nullptr, nullptr, 0, (int64_t)(unit - b.unit0[i]));
}

// Whether a launch of `kernel`, a quantizer that waits for what is in front of it, should begin before that has ended.  Eagerly:
// yes.  In a capture only behind one other kernel that nothing else follows yet: a graph runs a node that begins early in one
// line with the node in front, so that work prepared on a side branch (one quantizer behind the other, FCs behind each of them)
// would wait for the FCs beside it.  (Four quantizers beside four FC launches 121.6 -> 112.6 us; in one line with them 126 as
// without this rule, never early 129 and, as the decode FCs' own quantizers too, 4 rows x 4096 x 4096 7.6 -> 8.1.  It takes the
// host 0.15 us a launch; the look-up and the other quantizers do without it.)
bool begins_early(cudaStream_t s, const void* kernel) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    const cudaGraphNode_t* front = nullptr;
    const cudaGraphEdgeData* edges = nullptr;
    size_t n = 0, followers = 0;
    cudaGraphNodeType type = cudaGraphNodeTypeEmpty;
    cudaKernelNodeParams node = {};
    // (an error here is not the caller's; what there is to say about the stream the launch itself will say)
    if (cudaStreamGetCaptureInfo_v3(s, &status, nullptr, nullptr, &front, &edges, &n) != cudaSuccess) {
        cudaGetLastError();
        return true;
    }
    if (status != cudaStreamCaptureStatusActive) return true;
    if (n != 1) return false;
    if (cudaGraphNodeGetType(front[0], &type) != cudaSuccess ||
        cudaGraphNodeGetDependentNodes_v2(front[0], nullptr, nullptr, &followers) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    if (type != cudaGraphNodeTypeKernel || followers != 0) return false;
    if (cudaGraphKernelNodeGetParams(front[0], &node) != cudaSuccess) cudaGetLastError();  // (a kernel of another library)
    return node.func != kernel;
}

}  // namespace

int launch_quant_x_pre_batch(const q4fc_xq_call* calls, int n, int G, bool want_isum, bool pdl, cudaStream_t s) {
    QuantBatch b = {};
    int units = 0;
    for (int i = 0; i < n; i++) {
        const q4fc_xq_call& c = calls[i];
        if (c.rows == 0) continue;
        const int64_t Kg = (c.K + G - 1) / G;
        const int64_t chunks = (Kg * G + 127) / 128;
        uint8_t* base = static_cast<uint8_t*>(c.xq);
        const int k = b.n++;
        b.x[k] = c.x, b.rows[k] = (int)c.rows, b.K[k] = c.K, b.ldx[k] = c.ldx;
        b.codes[k] = reinterpret_cast<int8_t*>(base);
        b.sc[k] = reinterpret_cast<float*>(base + align_up((size_t)(c.rows * Kg * G), 256));
        b.vec_ok[k] = (c.K % 4 == 0) && (c.ldx % 4 == 0) && ((reinterpret_cast<uintptr_t>(c.x) & 15) == 0);
        b.unit0[k] = units;
        if (chunks * c.rows > 0x3fffffff - units) {
            set_error("quant_x_q8_batch: too many values for one launch");
            return Q4FC_ELIMIT;
        }
        units += (int)(chunks * c.rows);
    }
    if (b.n == 0) return Q4FC_OK;
    b.unit0[b.n] = units;
    auto* kernel = G == 32 ? quant_x_pre_batch_kernel<32> : quant_x_pre_batch_kernel<128>;
    // (it waits before it reads, and without `pdl` releases the FC only after that)
    DependentLaunch l(dim3((unsigned)((units + 3) / 4)), 128, s, pdl || begins_early(s, reinterpret_cast<const void*>(kernel)));
    Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, kernel, b, (int)want_isum, (int)pdl));
    return Q4FC_OK;
}

size_t quant_pre_bytes(int64_t rows, int64_t K, int G) {
    const int64_t Kg = (K + G - 1) / G;
    return align_up((size_t)(rows * Kg * G), 256) + align_up((size_t)Kg * 16 * sizeof(float), 256);
}

int launch_quant_x_pre(const float* x, int rows, int64_t K, int64_t ldx, int G, bool want_isum, int8_t* codes,
                       float* sc, bool pdl, cudaStream_t s, const float* up, float* prod, int64_t ldp) {
    const int64_t Kg = (K + G - 1) / G;
    const int64_t chunks = (Kg * G + 127) / 128;
    const int64_t grid = (chunks * rows + 3) / 4;
    const int vec_ok = (K % 4 == 0) && (ldx % 4 == 0) && ((reinterpret_cast<uintptr_t>(x) & 15) == 0) &&
                       ((reinterpret_cast<uintptr_t>(up) & 15) == 0);
    auto* kernel = G == 32 ? quant_x_pre_kernel<32> : quant_x_pre_kernel<128>;
    // (it waits before it reads, and without `pdl` releases the FC only after that)
    DependentLaunch l(dim3((unsigned)grid), 128, s, pdl || begins_early(s, reinterpret_cast<const void*>(kernel)));
    Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, kernel, x, rows, K, ldx, Kg, vec_ok, (int)want_isum, (int)pdl, codes, sc, up, prod, ldp));
    return Q4FC_OK;
}

int launch_quant_x_tile(const float* x, int64_t rows, int64_t K, int64_t ldx, int G, bool sums, int tile, bool f16,
                        int8_t* codes, float* sc, cudaStream_t s) {
    const int64_t Kg = (K + G - 1) / G;
    if (rows == 0 || Kg == 0) return Q4FC_OK;
    const int64_t chunks = (Kg * G + 127) / 128;
    const bool many = rows * chunks >= kManyUnits;
    const int64_t grid = (rows + kQxWarps - 1) / kQxWarps * (many ? (chunks + kManyChunks - 1) / kManyChunks : chunks);
    if (grid > 0x7fffffffLL) {
        set_error("quant_x: %lld x %lld exceeds the grid limit", (long long)rows, (long long)K);
        return Q4FC_ELIMIT;
    }
    const int vec_ok = (K % 4 == 0) && (ldx % 4 == 0) && ((reinterpret_cast<uintptr_t>(x) & 15) == 0);
    const int l2 = tile == 128 ? 7 : 6;
    DependentLaunch l(dim3((unsigned)grid), kQxWarps * 32, s);
    auto launch = [&](auto n) -> int {
        constexpr int N = decltype(n)::value;
        auto* kernel = G == 128 ? quant_x_tile_kernel<128, false, N> : f16 ? quant_x_tile_kernel<32, true, N> : quant_x_tile_kernel<32, false, N>;
        Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, kernel, x, rows, K, ldx, Kg, vec_ok, (int)sums, l2, codes, sc));
        return Q4FC_OK;
    };
    return many ? launch(std::integral_constant<int, kManyChunks>{}) : launch(std::integral_constant<int, 1>{});
}

int launch_quant_x_group(const GroupQuant& q, int G, bool f16, cudaStream_t s) {
    if (q.rows == 0) return Q4FC_OK;
    const int64_t chunks = (q.Kg * G + 127) / 128;
    const int64_t x_rows = q.rows / q.per_row;
    const bool many = x_rows * chunks >= kManyUnits;
    const int64_t grid = (x_rows + kQxWarps - 1) / kQxWarps * (many ? (chunks + kManyChunks - 1) / kManyChunks : chunks);
    if (grid > 0x7fffffffLL) {
        set_error("quant_x: %lld x %lld exceeds the grid limit", (long long)q.rows, (long long)q.K);
        return Q4FC_ELIMIT;
    }
    DependentLaunch l(dim3((unsigned)grid), kQxWarps * 32, s);
    auto launch = [&](auto n) -> int {
        constexpr int N = decltype(n)::value;
        auto* kernel = G == 128 ? quant_x_group_kernel<128, false, N> : f16 ? quant_x_group_kernel<32, true, N> : quant_x_group_kernel<32, false, N>;
        Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, kernel, q));
        return Q4FC_OK;
    };
    return many ? launch(std::integral_constant<int, kManyChunks>{}) : launch(std::integral_constant<int, 1>{});
}

int launch_quant_x(const float* x, int64_t rows, int64_t K, int64_t ldx, int G, float scale, int8_t* codes,
                   float* scales, float* gsums, cudaStream_t s) {
    const int64_t Kg = (K + G - 1) / G;
    if (rows == 0 || Kg == 0) return Q4FC_OK;
    const int64_t chunks = (Kg * G + 127) / 128;
    const int64_t grid = (rows * chunks + kQxWarps - 1) / kQxWarps;
    if (grid > 0x7fffffffLL) {
        set_error("quant_x: %lld x %lld exceeds the grid limit", (long long)rows, (long long)K);
        return Q4FC_ELIMIT;
    }
    const int vec_ok = (K % 4 == 0) && (ldx % 4 == 0) && ((reinterpret_cast<uintptr_t>(x) & 15) == 0);
    auto* kernel = G == 32 ? quant_x_kernel<32> : quant_x_kernel<128>;
    DependentLaunch l(dim3((unsigned)grid), kQxWarps * 32, s);
    Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, kernel, x, rows, K, ldx, Kg, scale, vec_ok, codes, scales, gsums));
    return Q4FC_OK;
}

}  // namespace q4fc
