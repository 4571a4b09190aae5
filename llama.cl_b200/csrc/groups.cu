// Rows grouped by an id, and the router in front of a layer of experts.  No counterpart in the reference, whose every FC
// gives all rows the same weights (ops/op_fc.hpp:286-426).
//
//   route:  p = softmax(logits) over the experts of a token; its top_k largest, the lowest index first where they are
//           equal; an expert whose logit is -inf is closed and never chosen (id -1, weight 0 where none is left).
//           Weights p, or p over the sum of the chosen ones.  The choice compares logits, no exponentials.
//   group:  a stable counting sort of the (token, slot) pairs by expert, or of rows by adapter (groups.cuh).
//
// Route: a warp per token, a lane holds every 32nd logit.  A step of the choice is two warp reductions, of the largest key
// and of the lowest index that has it; only the winner looks for its next.
// Group, up to 256 rows: one CTA, a thread per row, that counts the rows in front of its own: those with a lower id and
// those with the same that come earlier.  All else follows from these two numbers.
// Group, more rows: one cluster.  Each warp owns a contiguous piece of the rows and its own bins in shared memory, so that
// equal ids need no atomics whose order would decide places: it counts its piece (lanes with equal ids find one another with
// ballots, the first adds) and notes each row's place among its own; the bins of all warps and CTAs are summed in order
// and give the places in front.  The same from run to run.
//
// Bound by the latencies of one CTA's (or cluster's) steps, not by bytes.  Measured, one call behind another: route, 1 token of 8 experts
// 2.5 us, 8 of 64 3.6, 333 of 64 7.8 (two launches), 4096 of 128, 8 each, 15.2; group, 48 rows 2.5, 2048 rows 6.5 (by one CTA 7.7).
#include <cooperative_groups.h>

#include <atomic>
#include <type_traits>

#include "groups.cuh"

namespace cg = cooperative_groups;

namespace q4fc {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kCluster = 8;               // CTAs that share a long list
constexpr uint32_t kClosed = 0x007fffffu;  // key of -inf; finite numbers are above

// order-preserving, -0 and 0 equal; NaN below everything
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 0u : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

struct RouteArgs {
    const float* logits;
    int64_t tokens, ld;
    int experts, top_k, renormalize;
    float* weights;
    int32_t* ids;
};

// One token, by one warp; NV logits a lane.
template <int NV>
__device__ __forceinline__ void route_token(const RouteArgs& a, int64_t token, int lane) {
    const float* src = a.logits + token * a.ld;
    uint32_t key[NV];
    bool nan = false;
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int e = lane + 32 * i;
        const float x = e < a.experts ? ld_after_wait(src + e) : -INFINITY;
        key[i] = key_of(x);
        nan |= x != x;
        best = max(best, key[i]);
    }
    nan = __any_sync(0xffffffffu, nan);
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const float most = value_of(top);
    float total = 0.0f;
    if (!a.renormalize && top > kClosed) {
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (key[i] >= kClosed) total += expf(value_of(key[i]) - most);  // (-inf: 0)
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    }
    int id = -1;       // of slot `lane`
    float mine = 0.0f;
    for (int s = 0; s < a.top_k; s++) {
        const uint32_t k = __reduce_max_sync(0xffffffffu, best);
        if (k <= kClosed) break;
        int at = 0x7fffffff;
        if (best == k) {
#pragma unroll
            for (int i = NV - 1; i >= 0; i--)
                if (key[i] == k) at = lane + 32 * i;
        }
        at = __reduce_min_sync(0xffffffffu, (unsigned)at);
        const float w = expf(value_of(k) - most);
        if (a.renormalize) total += w;
        if (lane == s) id = at, mine = w;
        if (lane == (at & 31)) {
            best = 0;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                if (i == at >> 5) key[i] = 0;
                best = max(best, key[i]);
            }
        }
    }
    if (lane < a.top_k) {
        a.ids[token * a.top_k + lane] = id;
        a.weights[token * a.top_k + lane] = nan ? __uint_as_float(0x7fc00000u) : id < 0 ? 0.0f : __fdiv_rn(mine, total);
    }
}

template <int NV>
__global__ void __launch_bounds__(256) route_kernel(const RouteArgs a) {
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    const int64_t token = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (token < a.tokens) route_token<NV>(a, token, threadIdx.x & 31);
}

struct GroupArgs {
    const void* ids;
    int i32;
    int64_t rows, piece;  // rows of a warp
    int n;
    GroupPlan plan;
    int* status;
};
__device__ __forceinline__ int bin_of(const GroupArgs& a, int64_t i) {
    const int64_t id = a.i32 ? (int64_t)__ldcg(static_cast<const int*>(a.ids) + i) : (int64_t)__ldcg(static_cast<const long long*>(a.ids) + i);
    if (id >= a.n) atomicOr(a.status, kStatusBadGroup);
    return id >= 0 && id < a.n ? (int)id : a.n;
}

// Up to kFew rows.  NV > 0: the warps choose the experts of the tokens first (NV logits a lane).
constexpr int kFew = 256;
template <int NV>
__global__ void __launch_bounds__(kFew) group_few_kernel(const GroupArgs a, const RouteArgs route) {
    __shared__ __align__(16) int bins[kFew], sorted[kFew];
    __shared__ int tiles_to[kTileSizes][kFew + 1];  // tiles that begin in front of a place
    __shared__ int warp_tiles[kTileSizes][kFew / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, me = threadIdx.x, rows = (int)a.rows;
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    if constexpr (NV > 0) {
        for (int64_t t = warp; t < route.tokens; t += kFew / 32) route_token<NV>(route, t, lane);
        __syncthreads();
    }
    const int b = me < rows ? bin_of(a, me) : a.n + 1;  // (behind all that are there)
    bins[me] = b;
    __syncthreads();
    int less = 0, before = 0, equal = 0;
    for (int i = 0; i < rows; i += 4) {
        const int4 o = *reinterpret_cast<const int4*>(bins + i);
        less += (o.x < b) + (o.y < b) + (o.z < b) + (o.w < b);
        equal += (o.x == b) + (o.y == b) + (o.z == b) + (o.w == b);
        before += (o.x == b && i < me) + (o.y == b && i + 1 < me) + (o.z == b && i + 2 < me) + (o.w == b && i + 3 < me);
    }
    const int place = me < rows ? less + before : me;
    sorted[place] = b;
    // a tile of a size begins at this row's place
    for (int j = 0; j < kTileSizes; j++) tiles_to[j][place] = b < a.n && before % tile_rows(j) == 0;
    if (me < rows) a.plan.order[place] = me, a.plan.group_of[me] = b, a.plan.place_of[me] = place;
    __syncthreads();
    // (place me) tiles in front
    int begins[kTileSizes], in_warp[kTileSizes];
#pragma unroll
    for (int j = 0; j < kTileSizes; j++) {
        begins[j] = tiles_to[j][me];
        const uint32_t mask = __ballot_sync(0xffffffffu, begins[j]);
        in_warp[j] = __popc(mask & ((1u << lane) - 1));
        if (lane == 0) warp_tiles[j][warp] = __popc(mask);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kTileSizes; j++) {
        int front = in_warp[j], all = 0;
#pragma unroll
        for (int w = 0; w < kFew / 32; w++) {
            const int c = warp_tiles[j][w];
            if (w < warp) front += c;
            all += c;
        }
        tiles_to[j][me] = front;
        if (me == 0) tiles_to[j][kFew] = all;
    }
    if (me < 16) {
        int all = 0;
        if (me < kTileSizes)
            for (int w = 0; w < kFew / 32; w++) all += warp_tiles[me][w];
        a.plan.counts[me] = all;
    }
    __syncthreads();
    if (b < a.n)
        for (int j = 0; j < kTileSizes; j++)
            if (before % tile_rows(j) == 0) a.plan.tiles[j][tiles_to[j][place]] = make_int4(b, place, min(tile_rows(j), equal - before), 0);
    for (int e = me; e <= a.n; e += kFew) {  // the first place of a group
        int lo = 0, hi = rows;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (sorted[mid] < e) lo = mid + 1; else hi = mid;
        }
        a.plan.offsets[e] = lo;
        for (int j = 0; j < kTileSizes; j++) a.plan.tile0[j][e] = tiles_to[j][lo];
    }
}

// More rows.
constexpr int kHeld = 8;  // sets of 32 rows of a warp that stay in registers between its two walks
constexpr int kStaged = kWarps * kHeld * 32;  // rows of a CTA that are sorted in shared memory on their way out
constexpr int kScans = 2 + kTileSizes;  // rows of the groups, their tiles, this CTA's rows
__global__ void __launch_bounds__(kThreads, 1) group_kernel(const GroupArgs a) {
    extern __shared__ uint32_t bins[];  // [warp][n + 1]
    __shared__ uint32_t sums[kMaxGroups + 1];             // this CTA's rows of each group
    __shared__ uint32_t first[kMaxGroups + 1];            // its first place of each group
    __shared__ uint32_t start[kMaxGroups + 1];            // the group's first place
    __shared__ uint32_t here[kMaxGroups + 1];             // and the first among this CTA's rows
    __shared__ int tile0[kTileSizes][kMaxGroups + 1];     // first tile of each group
    __shared__ uint32_t warp_sum[kScans][kWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster.block_rank();
    const int nb = a.n + 1;  // bins; the last one is of rows without a group
    uint32_t* mine = bins + warp * nb;
    for (int i = lane; i < nb; i += 32) mine[i] = 0;
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    const int64_t begin = min(a.rows, ((int64_t)rank * kWarps + warp) * a.piece), end = min(a.rows, begin + a.piece);
    __syncwarp();
    // 32 rows: their bins, and the place of each among the warp's rows of its bin.  (Lanes with equal bins find one another bit by
    // bit: a match.any takes the longer the more different ones there are.)
    const int bits = 32 - __clz(a.n);
    auto count = [&](int b, bool there) {
        uint32_t same = __ballot_sync(0xffffffffu, there);
        for (int i = 0; i < bits; i++) {
            const uint32_t set = __ballot_sync(0xffffffffu, (b >> i) & 1);
            same &= (b >> i) & 1 ? set : ~set;
        }
        const uint32_t below = same & ((1u << lane) - 1);
        const uint32_t at = there ? mine[b] : 0;
        __syncwarp();
        if (there && below == 0) mine[b] = at + __popc(same);
        __syncwarp();
        return at + __popc(below);
    };
    int held[kHeld];
    uint32_t local[kHeld];
#pragma unroll
    for (int h = 0; h < kHeld; h++) held[h] = begin + 32 * h + lane < end ? bin_of(a, begin + 32 * h + lane) : -1;
#pragma unroll
    for (int h = 0; h < kHeld; h++)
        if (begin + 32 * h < end) local[h] = count(held[h], held[h] >= 0);
    for (int64_t i0 = begin + 32 * kHeld; i0 < end; i0 += 32) {
        const bool there = i0 + lane < end;
        count(there ? bin_of(a, i0 + lane) : -1, there);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < nb; b += kThreads) {  // warps in order
        uint32_t c[kWarps], sum = 0;
#pragma unroll
        for (int w = 0; w < kWarps; w++) c[w] = bins[w * nb + b];
#pragma unroll
        for (int w = 0; w < kWarps; w++) bins[w * nb + b] = sum, sum += c[w];
        sums[b] = sum;
    }
    cluster.sync();
    // group b = threadIdx.x (kMaxGroups = kThreads of them): its rows, those of the CTAs in front, its first place and tiles; by the warps
    // that have any
    const int group_warps = (a.n + 31) / 32;
    uint32_t all = 0, front = 0;
    uint32_t v[kScans], own[kScans];
    if (warp < group_warps) {
        if ((int)threadIdx.x < a.n)
            for (int c = 0; c < kCluster; c++) {
                const uint32_t v = cluster.map_shared_rank(sums, c)[threadIdx.x];
                all += v;
                if (c < rank) front += v;
            }
        v[0] = all, v[1 + kTileSizes] = (int)threadIdx.x < a.n ? sums[threadIdx.x] : 0;
#pragma unroll
        for (int j = 0; j < kTileSizes; j++) v[1 + j] = (all + tile_rows(j) - 1) / tile_rows(j);
#pragma unroll
        for (int j = 0; j < kScans; j++) own[j] = v[j];
#pragma unroll 1
        for (int off = 1; off < 32; off <<= 1)
#pragma unroll
            for (int j = 0; j < kScans; j++) {
                const uint32_t o = __shfl_up_sync(0xffffffffu, v[j], off);
                if (lane >= off) v[j] += o;
            }
        if (lane == 31)
#pragma unroll
            for (int j = 0; j < kScans; j++) warp_sum[j][warp] = v[j];
    }
    __syncthreads();
    if (warp < group_warps) {
        uint32_t total[kScans];
#pragma unroll
        for (int j = 0; j < kScans; j++) {
            const uint32_t w = lane < group_warps ? warp_sum[j][lane] : 0;
            total[j] = __reduce_add_sync(0xffffffffu, w);
            v[j] += __reduce_add_sync(0xffffffffu, lane < warp ? w : 0u) - own[j];  // in front of this group
        }
        if ((int)threadIdx.x < a.n) {
            first[threadIdx.x] = v[0] + front, start[threadIdx.x] = v[0], here[threadIdx.x] = v[1 + kTileSizes];
#pragma unroll
            for (int j = 0; j < kTileSizes; j++) tile0[j][threadIdx.x] = (int)v[j + 1];
            if (rank == 0) {
                a.plan.offsets[threadIdx.x] = (int)v[0];
#pragma unroll
                for (int j = 0; j < kTileSizes; j++) a.plan.tile0[j][threadIdx.x] = (int)v[j + 1];
            }
        }
        if (threadIdx.x == 0) {
            uint32_t none_front = 0;  // of rows without a group
            for (int c = 0; c < rank; c++) none_front += cluster.map_shared_rank(sums, c)[a.n];
            first[a.n] = total[0] + none_front, start[a.n] = total[0], here[a.n] = total[1 + kTileSizes];
#pragma unroll
            for (int j = 0; j < kTileSizes; j++) tile0[j][a.n] = (int)total[j + 1];
            if (rank == 0) {
                a.plan.offsets[a.n] = (int)total[0];
#pragma unroll
                for (int j = 0; j < kTileSizes; j++) a.plan.tile0[j][a.n] = (int)total[j + 1];
#pragma unroll
                for (int j = 0; j < 16; j++) a.plan.counts[j] = j < kTileSizes ? (int)total[j + 1] : 0;
            }
        }
    }
    __syncthreads();
    // The rows' places.  A CTA's rows go through shared memory, in their order, if they fit: neighbours in it mostly are
    // neighbours in the plan (stored one by one, 32768 rows take 8 us more: a sector each).
    if (a.piece <= 32 * kHeld) {
        uint32_t* row_of = bins + kWarps * nb;
        uint16_t* bin_at = reinterpret_cast<uint16_t*>(row_of + kStaged);
#pragma unroll
        for (int h = 0; h < kHeld; h++)
            if (held[h] >= 0) {
                const uint32_t at = here[held[h]] + mine[held[h]] + local[h];
                const int64_t i = begin + 32 * h + lane;
                row_of[at] = (uint32_t)i, bin_at[at] = (uint16_t)held[h];
                a.plan.group_of[i] = held[h], a.plan.place_of[i] = (int)(first[held[h]] + at - here[held[h]]);
            }
        __syncthreads();
        const uint32_t there = here[a.n] + sums[a.n];
        for (uint32_t i = threadIdx.x; i < there; i += kThreads) {
            const int b = bin_at[i];
            const uint32_t place = first[b] + i - here[b];
            a.plan.order[place] = (int)row_of[i];
        }
    } else {
        for (int64_t i0 = begin; i0 < end; i0 += 32) {
            const bool there = i0 + lane < end;
            const int b = there ? bin_of(a, i0 + lane) : -1;
            const uint32_t local = count(b, there);
            if (there) {
                const uint32_t place = first[b] + local;
                a.plan.order[place] = (int)(i0 + lane), a.plan.group_of[i0 + lane] = b, a.plan.place_of[i0 + lane] = (int)place;
            }
        }
    }
    // tiles of all sizes, one list: the group of tile i of a size is the last whose first tile is not behind it
    int ends[kTileSizes];
#pragma unroll
    for (int j = 0; j < kTileSizes; j++) ends[j] = (j > 0 ? ends[j - 1] : 0) + tile0[j][a.n];
    for (int at = rank * kThreads + threadIdx.x; at < ends[kTileSizes - 1]; at += kCluster * kThreads) {
        int j = 0, i = at;
#pragma unroll
        for (int k = 0; k + 1 < kTileSizes; k++)
            if (at >= ends[k]) j = k + 1, i = at - ends[k];
        int lo = 0, hi = a.n;  // tile0[lo] <= i < tile0[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (tile0[j][mid] <= i) lo = mid; else hi = mid;
        }
        const int size = tile_rows(j), in = (i - tile0[j][lo]) * size;
        a.plan.tiles[j][i] = make_int4(lo, (int)start[lo] + in, min(size, (int)(start[lo + 1] - start[lo]) - in), 0);
    }
    cluster.sync();  // nobody leaves while its sums are being read
}

template <int NV>
int launch_group_few(const GroupArgs& a, const RouteArgs& route, cudaStream_t s) {
    DependentLaunch l(dim3(1), kFew, s);
    Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, group_few_kernel<NV>, a, route));
    return Q4FC_OK;
}
int launch_group(const GroupArgs& a, cudaStream_t s) {
    static std::atomic<bool> attr_done[64] = {};  // set once per device; a second setter repeats the same call
    auto* fn = group_kernel;
    const size_t most = kWarps * (kMaxGroups + 1) * sizeof(uint32_t) + kStaged * 6;
    int dev = 0;
    Q4FC_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr_done[dev]) {
        Q4FC_CUDA_OK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
        if (dev < 64) attr_done[dev] = true;
    }
    DependentLaunch l(dim3(kCluster), kThreads, s);
    cudaLaunchAttribute attrs[2] = {l.attr, {}};
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = kCluster, attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    l.cfg.attrs = attrs, l.cfg.numAttrs = 2;
    l.cfg.dynamicSmemBytes = kWarps * (size_t)(a.n + 1) * sizeof(uint32_t) + kStaged * 6;
    Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, fn, a));
    return Q4FC_OK;
}
// NV: logits a lane holds, for as many experts
template <typename F>
int with_lanes(int experts, F f) {
    if (experts <= 32) return f(std::integral_constant<int, 1>{});
    if (experts <= 64) return f(std::integral_constant<int, 2>{});
    if (experts <= 128) return f(std::integral_constant<int, 4>{});
    if (experts <= 256) return f(std::integral_constant<int, 8>{});
    return f(std::integral_constant<int, 32>{});
}
int group_args(GroupArgs* a, const void* ids, int i32, int64_t rows, int64_t n, void* groups) {
    a->ids = ids, a->i32 = i32, a->rows = rows, a->n = (int)n, a->plan = group_plan(groups, rows, n);
    constexpr int64_t warps = (int64_t)kCluster * kWarps;
    a->piece = (rows + warps - 1) / warps;
    a->status = ring_status_word();
    return a->status ? Q4FC_OK : Q4FC_ECUDA;
}

}  // namespace

int launch_group_rows(const void* ids, int ids_are_i32, int64_t rows, int64_t n, void* groups, cudaStream_t s) {
    GroupArgs a = {};
    if (int rc = group_args(&a, ids, ids_are_i32, rows, n, groups)) return rc;
    if (rows <= kFew) return launch_group_few<0>(a, RouteArgs{}, s);
    return launch_group(a, s);
}

int launch_route_top_k(const float* logits, int64_t tokens, int64_t experts, int64_t ld, int64_t top_k, int renormalize,
                       float* weights, int32_t* ids, void* groups, cudaStream_t s) {
    RouteArgs route = {logits, tokens, ld, (int)experts, (int)top_k, renormalize, weights, ids};
    GroupArgs a = {};
    const int64_t rows = tokens * top_k;
    if (int rc = group_args(&a, ids, 1, rows, experts, groups)) return rc;
    return with_lanes((int)experts, [&](auto nv) {
        constexpr int NV = decltype(nv)::value;
        // (a token for each warp of the plan's launch: 8 of 64 experts, 6 each, 3.6 us; 16 of them, 8 each, 6.2 so and 5.4 in two launches)
        if (rows <= kFew && tokens <= kFew / 32) return launch_group_few<NV>(a, route, s);
        DependentLaunch l(dim3((unsigned)((tokens + 7) / 8)), 256, s);
        Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, route_kernel<NV>, route));
        return rows <= kFew ? launch_group_few<0>(a, RouteArgs{}, s) : launch_group(a, s);
    });
}

}  // namespace q4fc
