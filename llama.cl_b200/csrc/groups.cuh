// Rows grouped by an id: what the kernels whose weights depend on the row (experts, adapters) read of a plan that
// groups.cu makes.  A plan is one device buffer of int32:
//   [0, 16)        tiles of 8, 16, 64 and 128 rows in use; the others 0
//   offsets[n + 1] first place in `order` of each group; offsets[n]: of the rows without one
//   order[rows]    row numbers, sorted by group and stable: the grouped ones, then those without a group
//   tiles          of 8, 16, 64 and 128 rows: {group, first place in order, rows, 0}; a tile's rows are of one group
//   group_of[rows] the group of each row (n: none)
//   place_of[rows] the place of each row in order
//   tile0[n + 1]   of 8, 16, 64 and 128 rows: the first tile of each group
// Each part starts on 16 bytes.  No group has more tiles than its rows / size + 1, so rows / size + min(n, rows) places are enough.
#pragma once
#include "common.cuh"

namespace q4fc {

constexpr int64_t kMaxGroups = 1024;       // bins of a warp in shared memory
constexpr int64_t kMaxGroupRows = 1 << 23;
enum { kTiles8, kTiles16, kTiles64, kTiles128, kTileSizes };
__host__ __device__ constexpr int tile_rows(int which) { return which == kTiles8 ? 8 : which == kTiles16 ? 16 : which == kTiles64 ? 64 : 128; }

struct GroupPlan {
    int* counts;        // tiles in use, by size
    int* offsets;
    int* order;
    int4* tiles[kTileSizes];
    int *group_of, *place_of;
    int* tile0[kTileSizes];
    int64_t bytes;
};
__host__ __device__ inline int64_t most_tiles(int which, int64_t rows, int64_t n) {
    return rows / tile_rows(which) + (n < rows ? n : rows);
}
inline GroupPlan group_plan(void* buffer, int64_t rows, int64_t n) {
    GroupPlan p;
    int64_t at = 64;
    uint8_t* base = static_cast<uint8_t*>(buffer);
    auto take = [&](int64_t bytes) {
        uint8_t* r = base ? base + at : nullptr;
        at += (bytes + 15) / 16 * 16;
        return r;
    };
    p.counts = reinterpret_cast<int*>(base);
    p.offsets = reinterpret_cast<int*>(take((n + 1) * 4));
    p.order = reinterpret_cast<int*>(take(rows * 4));
    for (int w = 0; w < kTileSizes; w++) p.tiles[w] = reinterpret_cast<int4*>(take(most_tiles(w, rows, n) * 16));
    p.group_of = reinterpret_cast<int*>(take(rows * 4));
    p.place_of = reinterpret_cast<int*>(take(rows * 4));
    for (int w = 0; w < kTileSizes; w++) p.tile0[w] = reinterpret_cast<int*>(take((n + 1) * 4));
    p.bytes = at;
    return p;
}

// groups.cu
int launch_group_rows(const void* ids, int ids_are_i32, int64_t rows, int64_t n, void* groups, cudaStream_t s);
int launch_route_top_k(const float* logits, int64_t tokens, int64_t experts, int64_t ld, int64_t top_k, int renormalize,
                       float* weights, int32_t* ids, void* groups, cudaStream_t s);

// The experts' product (fc_experts.cu and what it launches).
struct GroupQuant {  // quant_x.cu
    const float* x;
    int64_t rows, K, Kg, ldx;  // rows: pairs of the plan
    int64_t per_row;           // pairs that share a row of x
    const int *group_of, *place_of, *offsets, *tile0;
    int n, log2tile, vec_ok, gated, sums, isum;
    int8_t* codes;
    float* sc;
    float* y;                  // [rows][ldy]: rows without an expert are zeroed
    int64_t N, ldy;
};
int launch_quant_x_group(const GroupQuant& q, int G, bool f16, cudaStream_t s);

struct ExpertsCall {
    const float* x;
    int64_t rows, K, ldx, per_row;  // pairs; pairs that share a row of x
    bool gated;
    const uint8_t* wq;              // [n][Ng][Kg][block]
    int64_t Ng, Kg;
    int qtype, G;
    int64_t N;
    GroupPlan plan;
    int64_t n, most_rows;           // experts; no expert has more pairs
    float* y;                       // [rows][ldy], in the order of the pairs
    int64_t ldy;
    unsigned flags;
    uint8_t* scratch;
};

size_t experts_gemm_scratch(int64_t rows, int64_t Kg, int G, int64_t n);  // fc_prefill.cu
int launch_experts_gemm(const ExpertsCall& c, GroupQuant q, cudaStream_t s);
// fc_experts_few.cu: experts with few rows
bool experts_few_serves(int64_t rows, int64_t Kg, int64_t Ng, int G, int64_t n);
size_t experts_few_scratch(int64_t rows, int64_t Kg, int G, int64_t n);
int launch_experts_few(const ExpertsCall& c, GroupQuant q, cudaStream_t s);
// fc_experts.cu; with weights [rows / top_k][top_k] c.y is [rows / top_k][ldy]
size_t experts_scratch_bytes(int64_t rows, int64_t K, int64_t N, int G, int64_t n, bool weighted);
int launch_fc_experts(ExpertsCall c, const float* weights, int64_t top_k, cudaStream_t s);

// lora.cu
struct LoraCall {
    const float* x;
    int64_t rows, K, ldx;
    const void *a, *b;   // [n][rank][K], [n][N][rank]
    int dtype;
    int64_t n, rank, N;
    const float* scales;
    GroupPlan plan;
    float* y;
    int64_t ldy;
    void* scratch;
};
size_t lora_scratch_bytes(int64_t rows, int64_t rank);
struct QuantPre;  // quant_pre.cuh
int launch_lora_add(const LoraCall& c, cudaStream_t s);
// around a decode FC (rows <= 8): in front of it, y of the adapters alone and the FC's quantized input
int launch_lora_first(const LoraCall& c, const QuantPre& q, cudaStream_t s);
// around a launch that computes y from x, between them: y is complete where what is in front of that launch is
int launch_lora_before(const LoraCall& c, cudaStream_t s);
int launch_lora_behind(const LoraCall& c, cudaStream_t s);

}  // namespace q4fc
