// FC by expert where experts have few rows: a weight-streaming kernel over the plan's tiles of up to 16 rows (groups.cuh).
// Per pair the arithmetic is that of fc_Q4A (ops/op_fc.hpp:286-426): exact integer products per K group, scaled in fp32.
//
// Work.  One CTA per SM, 16 warps.  (tiles in use) x (stripes of 32 columns) are one list, known on the device alone; a CTA
// takes a contiguous share of whole stripes, and its warps contiguous shares of the share's chunks (32 columns x 128 k, 2 to
// 2.5 KB): a warp walks through the ends of stripes as they come.  It has a ring of its own in shared memory, which its first
// lane fills with bulk copies, so no warp waits for another one until the end.  Sums of a stripe that one warp has walked
// whole go straight to y; the others (at most two a warp) meet in shared memory behind the one barrier and are added in
// warp order.  No atomics, the same from run to run.
//
// Why not the kernel of fc_decode_ring_impl.cuh, whose 16 warps share every stripe: a stripe of a narrow expert is one block for
// each of them, and meeting over it costs more than the block (K = 2048, group 128: 367 instructions per block, here about 110).
//
// Arithmetic.  mma.sync.m16n8k32 (u8 x s8), weight columns on the 16-row side, activations on the 8 columns.  Experts of a small
// batch mostly have one or two rows; eight columns for them would be scaled at the price of eight.  So the columns are shared by
// rows and K groups: with at most 2 rows four K groups in turn have two columns each, with at most 4 two groups have four --
// the codes of the other groups' columns are zeros -- and one pass of conversion and scaling, in which a lane has another
// group's scales, serves all four (or two).  Up to 16 rows are two sets of eight columns on weights that are unpacked once.
// Codes and scales come from global memory, through L1.
//
// Measured, with the quantizer in front: one token to two of 8 experts, 4096 x 22016, Q4_1 group 32: 113 MB in 22.4 to 23.3 us, 5 TB/s; 8 tokens
// to 6 of 64, 2048 x 2816, group 128: 28.2; 170 tokens to 6 of 64, 1408 x 2048, group 32: 48.4.  There the scaling, in fp32 for every row,
// column and K group, is the work: half an instruction a cycle and scheduler, fixed latencies first among the waits (fewer instructions alone
// changed nothing).
#include "decode_math.cuh"
#include "groups.cuh"
#include "ring_ptx.cuh"

#include <atomic>
#include <type_traits>

namespace q4fc {
namespace {

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kMaxDepth = 3;
constexpr int kMostTiles = 2 * kThreads;  // in shared memory
constexpr int kTileRows = 16;

struct FewParams {
    const int8_t* codes;  // [place][row_bytes]
    const float* sc;      // [tile][K group, whole chunks][two rows of 16][their scales, sums]
    const uint8_t* wq;
    float* y;
    const int4* tiles;
    const int *tile_count, *order;
    int64_t row_bytes, N, ldy, group_bytes;
    int Ng, Kg, chunks;  // chunks of a stripe
    int most_tiles, part_rows, depth, last_bytes, y_vec, weigh, part_off, ring_off;
    int* status;
};

__device__ __forceinline__ bool elect_lane() {  // one lane of a converged warp
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}

// What a chunk costs in a tile of at most 2, 4, 8 and 16 rows.  (64 experts x 1408 x 2048, group 32, all with as many rows: 28, 29, 30 and
// 42 us, of which other launches take 6 to 10.  170 tokens to 6 of them each: equal shares of the stripes 5 us more.)
__device__ constexpr int kCosts[4] = {6, 6, 7, 10};

template <int G, int QTYPE>
struct FewShape {
    static constexpr int BS = block_bytes(QTYPE, G);
    static constexpr int kBlocks = 128 / G;  // of a chunk
    static constexpr int kSlot = kBlocks * BS;
};

__device__ __noinline__ void wait_longer(uint32_t bar, uint32_t parity, volatile int* fail, int* status) {
    mbar_wait(bar, parity, fail, status, 0x4658504C);  // 'FXPL'
}

// A warp's ring.  A slot that has been read takes what comes next: of its stripes the weights follow one another in memory, up to the
// end of an expert's.
template <int G, int QTYPE>
struct WarpRing {
    using S = FewShape<G, QTYPE>;
    const uint8_t* slot;    // read next
    uint32_t at, bar;       // its address and barrier
    uint32_t parity;
    int n;                  // its number
    int left;               // chunks that are not asked for yet
    int in_stripe, in_tile; // chunks to the end of the stripe and of the expert's weights, from the next one that is asked for on
    int tile;
    const uint8_t* from;    // where it is

    // the next chunk into a slot
    __device__ __forceinline__ void ask(const FewParams& p, const int4* tiles) {
        uint32_t bytes = S::kSlot;
        if (--in_stripe == 0) in_stripe = p.chunks, bytes = p.last_bytes;
        if (elect_lane()) {
            mbar_expect_tx(bar, bytes);
            bulk_g2s(at, from, bytes, bar);
        }
        from += bytes, left--;
        if (--in_tile == 0 && left > 0) {
            in_tile = p.chunks * p.Ng, tile++;
            from = p.wq + tiles[tile].x * p.group_bytes;
        }
    }
    __device__ __forceinline__ void step(const FewParams& p) {
        slot += S::kSlot, at += S::kSlot, bar += 8;
        if (++n == p.depth) {
            n = 0, parity ^= 1;
            slot -= p.depth * S::kSlot, at -= p.depth * S::kSlot, bar -= 8 * p.depth;
        }
    }
    __device__ __forceinline__ void wait(const FewParams& p, volatile int* fail) {
        if (__builtin_expect(!mbar_try_wait(bar, parity), 0)) wait_longer(bar, parity, fail, p.status);
    }
    // the slot has been read by all lanes
    __device__ __forceinline__ void next(const FewParams& p, const int4* tiles) {
        __syncwarp();
        if (left > 0) ask(p, tiles);
        step(p);
    }
};

// 32 columns x 32 k of a block: the words of block rows t, columns 4g .. 4g + 3, as the two MMAs want them.  (Block rows are 128 bytes
// apart: two 64-bit loads whose halves swap with the parity of t, see fc_decode_ring_impl.cuh.)
__device__ __forceinline__ uint4 load_words(const uint8_t* row, int t) {
    const bool odd = t & 1;
    const uint2 u = *reinterpret_cast<const uint2*>(row + (odd ? 8 : 0));
    const uint2 v = *reinterpret_cast<const uint2*>(row + (odd ? 0 : 8));
    return make_uint4(odd ? v.x : u.x, odd ? v.y : u.y, odd ? u.x : v.x, odd ? u.y : v.y);
}

// Integers without conversion: an MMA that starts from the bits of 1.5 x 2^23 leaves those of 1.5 x 2^23 + I (|I| < 2^22).
constexpr int kIntBits = 0x4B400000;
constexpr float kInt = 12582912.0f;
// D(16x8, s32) = A(16x32, u8) * B(32x8, s8) + C
__device__ __forceinline__ void mma_from(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const int (&c)[4]) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ uint64_t pair(int lo, int hi) { return pair(__int_as_float(lo), __int_as_float(hi)); }
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// The sums of chunks [kc0, kc1) of a stripe.  SHARE: K groups that share the eight columns (4, 2 or 1); SETS: of eight columns.
// acc[s][c]: column 4g + c of two rows of set s; lane t: SHARE 4: rows 0, 1, K groups t mod 4; 2: rows 2 (t % 2) and one more, K
// groups t / 2 mod 2; 1: rows 2t, 2t + 1.  What columns of rows beyond the tile's hold is not used.
template <int G, int QTYPE, bool SIGNED, int SHARE, int SETS>
__device__ __forceinline__ void walk(const FewParams& p, const int4* tiles, WarpRing<G, QTYPE>& ring, volatile int* fail, int lane, int4 tile,
                                     int tile_index, int kc0, int kc1, uint64_t (&acc)[SETS][4]) {
    using S = FewShape<G, QTYPE>;
    constexpr int BS = S::BS, kRows = 8 / SHARE;  // rows of a set
    const int g = lane >> 2, t = lane & 3;
    const int b_group = g / kRows, b_row = g % kRows;                              // what column g is of
    const int d_group = t * SHARE / 4, d_row = 2 * (t % (4 / SHARE));              // what this lane's columns 2t, 2t + 1 are of
    const int8_t* codes[SETS];
#pragma unroll
    for (int s = 0; s < SETS; s++) codes[s] = p.codes + (int64_t)(tile.y + min(8 * s + b_row, tile.z - 1)) * p.row_bytes + kc0 * 128 + 32 * t;
    const float* sc = p.sc + ((int64_t)tile_index * p.chunks + kc0) * (S::kBlocks * 32) + 2 * d_row;
#pragma unroll
    for (int s = 0; s < SETS; s++)
#pragma unroll
        for (int c = 0; c < 4; c++) acc[s][c] = 0;
    int start[4];  // (kept: four registers that the first MMA of a round starts from)
#pragma unroll
    for (int i = 0; i < 4; i++) asm volatile("mov.b32 %0, %1;" : "=r"(start[i]) : "n"(kIntBits));
    const uint64_t minus = pair(-kInt, -kInt);
    // scaling of what the columns have gathered; low, up: [columns 4g, 4g + 1 | 4g + 2, 4g + 3][row of the MMA's half][rows]; x4: scales of
    // the lane's two rows, their sums
    auto finish = [&](const int (&low)[SETS][2][4], const int (&up)[SETS][2][4], uint2 wd, uint2 wm, const ulonglong2 (&x4)[SETS]) {
        const float2 wd01 = __half22float2(*reinterpret_cast<const __half2*>(&wd.x)), wd23 = __half22float2(*reinterpret_cast<const __half2*>(&wd.y));
        const float2 wm01 = __half22float2(*reinterpret_cast<const __half2*>(&wm.x)), wm23 = __half22float2(*reinterpret_cast<const __half2*>(&wm.y));
        const float wdf[4] = {wd01.x, wd01.y, wd23.x, wd23.y}, wmf[4] = {wm01.x, wm01.y, wm23.x, wm23.y};
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const uint64_t wd2 = pair(wdf[c], wdf[c]), wm2 = pair(wmf[c], wmf[c]);
#pragma unroll
            for (int s = 0; s < SETS; s++) {
                int l0 = low[s][c / 2][c % 2 * 2], l1 = low[s][c / 2][c % 2 * 2 + 1];
                if (SIGNED) {
                    const float2 eights = unpair(x4[s].y);
                    l0 -= __float_as_int(eights.x), l1 -= __float_as_int(eights.y);
                }
                uint64_t f = add2(pair(l0, l1), minus);
                // (group 128: upper nibbles stay in place, 16 times their value; all of it is below 2^24 and exact)
                if constexpr (G == 128)
                    f = fma2(add2(pair(up[s][c / 2][c % 2 * 2], up[s][c / 2][c % 2 * 2 + 1]), minus), pair(0.0625f, 0.0625f), f);
                acc[s][c] = fma2(mul2(wd2, x4[s].x), f, acc[s][c]);
                if (QTYPE == 1) acc[s][c] = fma2(wm2, x4[s].y, acc[s][c]);
            }
        }
    };
    auto scales_of = [&](int kb, ulonglong2 (&x4)[SETS]) {  // K group kb behind kc0
#pragma unroll
        for (int s = 0; s < SETS; s++) x4[s] = __ldca(reinterpret_cast<const ulonglong2*>(sc + kb * 32 + 16 * s));
    };
    auto codes_of = [&](int chunk, uint4 (&x)[SETS][2]) {  // this lane's of a chunk's four times 32 k
#pragma unroll
        for (int s = 0; s < SETS; s++) {
            const uint4* from = reinterpret_cast<const uint4*>(codes[s] + 128 * chunk);
            x[s][0] = __ldca(from), x[s][1] = __ldca(from + 1);
        }
    };
    if constexpr (G == 32) {
#pragma unroll 1
        for (int kc = kc0; kc < kc1; kc++) {
            const int n = p.Kg - 4 * kc;  // blocks that are there; of others the codes and scales are zeros
            uint4 x[SETS][2];
            codes_of(0, x);
            ring.wait(p, fail);
            const uint8_t* words = ring.slot + t * 128 + g * 16;
#pragma unroll
            for (int i = 0; i < 4 / SHARE; i++) {
                const int mine = i * SHARE + d_group;
                ulonglong2 x4[SETS];
                scales_of(mine, x4);
                const uint8_t* tail = ring.slot + mine * BS + 16 * G + g * 8;
                uint2 wd = *reinterpret_cast<const uint2*>(tail), wm = make_uint2(0u, 0u);
                if (QTYPE == 1) wm = *reinterpret_cast<const uint2*>(tail + 64);
                if (mine >= n) wd = wm = make_uint2(0u, 0u);  // (not what an earlier chunk has left there)
                int I[SETS][2][4];
#pragma unroll
                for (int h = 0; h < SHARE; h++) {
                    const int j = i * SHARE + h;
                    const uint4 q = load_words(words + j * BS, t);
                    uint32_t l[4] = {q.x & kNibMask, q.y & kNibMask, q.z & kNibMask, q.w & kNibMask};
                    uint32_t u[4] = {(q.x >> 4) & kNibMask, (q.y >> 4) & kNibMask, (q.z >> 4) & kNibMask, (q.w >> 4) & kNibMask};
                    if (SIGNED)
#pragma unroll
                        for (int k = 0; k < 4; k++) l[k] ^= 0x08080808u, u[k] ^= 0x08080808u;
#pragma unroll
                    for (int s = 0; s < SETS; s++) {
                        uint32_t b0 = j % 2 ? x[s][j / 2].z : x[s][j / 2].x, b1 = j % 2 ? x[s][j / 2].w : x[s][j / 2].y;
                        if (SHARE > 1 && b_group != h) b0 = b1 = 0;
                        if (h == 0) {
                            mma_from(I[s][0], l[0], l[1], u[0], u[1], b0, b1, start), mma_from(I[s][1], l[2], l[3], u[2], u[3], b0, b1, start);
                        } else {
                            mma_u8s8(I[s][0], l[0], l[1], u[0], u[1], b0, b1), mma_u8s8(I[s][1], l[2], l[3], u[2], u[3], b0, b1);
                        }
                    }
                }
                finish(I, I, wd, wm, x4);
            }
            sc += 4 * 32;
#pragma unroll
            for (int s = 0; s < SETS; s++) codes[s] += 128;
            ring.next(p, tiles);
        }
    } else {
        // One block a chunk: the groups that share columns are successive chunks, `n` of them (all SHARE in the loop below).
        auto round = [&](auto whole, int n) {
            uint4 x[SETS][2];
            ulonglong2 x4[SETS];
            uint2 wd = make_uint2(0u, 0u), wm = make_uint2(0u, 0u);
            int low[SETS][2][4], up[SETS][2][4];
            constexpr bool kWhole = decltype(whole)::value;
            if (kWhole || b_group < n) {
                codes_of(b_group, x);
            } else {
#pragma unroll
                for (int s = 0; s < SETS; s++) x[s][0] = x[s][1] = make_uint4(0u, 0u, 0u, 0u);
            }
            if (kWhole || d_group < n) {
                scales_of(d_group, x4);
            } else {
#pragma unroll
                for (int s = 0; s < SETS; s++) x4[s] = make_ulonglong2(0, 0);
            }
#pragma unroll
            for (int h = 0; h < SHARE; h++) {
                if (!kWhole && h >= n) break;
                ring.wait(p, fail);
                if (SHARE == 1 || d_group == h) {
                    const uint8_t* tail = ring.slot + 16 * G + g * 8;
                    wd = *reinterpret_cast<const uint2*>(tail);
                    if (QTYPE == 1) wm = *reinterpret_cast<const uint2*>(tail + 64);
                }
                const uint8_t* words = ring.slot + t * 128 + g * 16;
#pragma unroll
                for (int pr = 0; pr < 2; pr++) {  // two sets of 32 k: lower nibbles in one MMA, upper ones, in place, in another
                    const uint4 qa = load_words(words + 1024 * pr, t), qb = load_words(words + 1024 * pr + 512, t);
                    const uint32_t a[4] = {qa.x, qa.y, qa.z, qa.w}, b[4] = {qb.x, qb.y, qb.z, qb.w};
                    constexpr uint32_t kFlip = SIGNED ? 0x88888888u : 0u;
                    uint32_t la[4], lb[4], ua[4], ub[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        la[k] = (a[k] ^ kFlip) & kNibMask, lb[k] = (b[k] ^ kFlip) & kNibMask;
                        ua[k] = (a[k] ^ kFlip) & ~kNibMask, ub[k] = (b[k] ^ kFlip) & ~kNibMask;
                    }
#pragma unroll
                    for (int s = 0; s < SETS; s++) {
                        uint4 o = x[s][pr];
                        if (SHARE > 1 && b_group != h) o = make_uint4(0u, 0u, 0u, 0u);
                        if (h == 0 && pr == 0) {
                            mma_from(low[s][0], la[0], la[1], lb[0], lb[1], o.x, o.z, start), mma_from(low[s][1], la[2], la[3], lb[2], lb[3], o.x, o.z, start);
                            mma_from(up[s][0], ua[0], ua[1], ub[0], ub[1], o.y, o.w, start), mma_from(up[s][1], ua[2], ua[3], ub[2], ub[3], o.y, o.w, start);
                        } else {
                            mma_u8s8(low[s][0], la[0], la[1], lb[0], lb[1], o.x, o.z), mma_u8s8(low[s][1], la[2], la[3], lb[2], lb[3], o.x, o.z);
                            mma_u8s8(up[s][0], ua[0], ua[1], ub[0], ub[1], o.y, o.w), mma_u8s8(up[s][1], ua[2], ua[3], ub[2], ub[3], o.y, o.w);
                        }
                    }
                }
                ring.next(p, tiles);
            }
            finish(low, up, wd, wm, x4);
        };
        int kc = kc0;
#pragma unroll 1
        for (; kc + SHARE <= kc1; kc += SHARE) {
            round(std::true_type{}, SHARE);
#pragma unroll
            for (int s = 0; s < SETS; s++) codes[s] += 128 * SHARE;
            sc += 32 * SHARE;
        }
        if (SHARE > 1 && kc < kc1) round(std::false_type{}, kc1 - kc);
    }
}

template <int G, int QTYPE, bool SIGNED>
__global__ void __launch_bounds__(kThreads, 1) experts_few_kernel(const __grid_constant__ FewParams p) {
    using S = FewShape<G, QTYPE>;
    extern __shared__ __align__(128) uint8_t smem[];
    // barriers [warp][kMaxDepth] | failure flag, costs by warp | tiles | partial sums of each warp's first stripe [warp][rows][32] | rings
    // [warp][depth].  Those of its last stripe go where its ring was.
    constexpr int kFail = kWarps * kMaxDepth * 8;
    int4* const tiles = reinterpret_cast<int4*>(smem + kFail + 16 + kWarps * 4);
    auto part = [&](int w, bool last) {
        return reinterpret_cast<float*>(smem + (last ? p.ring_off + w * p.depth * S::kSlot : p.part_off + w * p.part_rows * 128));
    };
    volatile int* fail = reinterpret_cast<volatile int*>(smem + kFail);
    int* const by_warp = reinterpret_cast<int*>(smem + kFail + 16);  // costs of the tiles that a warp has loaded
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t bars = smem_u32(smem) + warp * kMaxDepth * 8;
    if (lane < p.depth) mbar_init(bars + 8 * lane, 1);
    if (threadIdx.x == 0) *fail = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    // The plan, and then the weights: the quantizer in front has let this launch begin only when what is in front of it was complete.
    const int count = __ldcg(p.tile_count);
    auto cost = [&](int rows) { return rows <= 2 ? kCosts[0] : rows <= 4 ? kCosts[1] : rows <= 8 ? kCosts[2] : kCosts[3]; };
    int4 two[2];  // of the tiles, this thread's (kMostTiles)
    int costs[2] = {0, 0}, all = 0;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int i = 2 * threadIdx.x + k;
        two[k] = i < p.most_tiles ? __ldcg(p.tiles + i) : make_int4(0, 0, 0, 0);
        two[k].z = min(two[k].z, p.part_rows);
        if (i < count) costs[k] = cost(two[k].z);
    }
    if (p.weigh) {  // the costs in front of each tile, of a chunk each
        int v = costs[0] + costs[1];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, v, off);
            if (lane >= off) v += o;
        }
        if (lane == 31) by_warp[warp] = v;
        __syncthreads();
        v -= costs[0] + costs[1];
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const int c = by_warp[w];
            all += c;
            if (w < warp) v += c;
        }
        two[0].w = __float_as_int((float)v), two[1].w = __float_as_int((float)(v + costs[0]));
    }
#pragma unroll
    for (int k = 0; k < 2; k++)
        if (2 * (int)threadIdx.x + k < p.most_tiles) tiles[2 * threadIdx.x + k] = two[k];
    __syncthreads();
    // The CTA's stripes and its warps' chunks: equal shares of the chunks, or where tiles cost the SM more than their bytes, of the
    // tiles' costs.  (Places in the list of costs are floats: all CTAs and warps round them alike, and upwards with the place.  With the
    // divisions of 64-bit integers, and the costs summed by one warp, this took 4 us.)
    const int C = p.chunks;
    int s0, r;
    int mine;  // first chunk of warp `lane`
    if (!p.weigh) {
        const int stripes = count * p.Ng, each = stripes / (int)gridDim.x, more = stripes - each * (int)gridDim.x, b = (int)blockIdx.x;
        s0 = each * b + min(b, more), r = each + (b < more);
        mine = (int)((int64_t)r * C * min(lane, kWarps) / kWarps);
    } else {
        auto front = [&](int tile) { return __int_as_float(tiles[tile].w); };
        auto tile_at = [&](float place, int lo, int hi) {  // of tiles [lo, hi) the last whose costs begin at or in front of a place
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (front(mid) <= place) lo = mid; else hi = mid;
            }
            return lo;
        };
        // of a tile's pieces the first one that begins at or behind a place
        auto piece_at = [&](float place, int tile, int pieces) {
            return min(pieces, (int)ceilf((place - front(tile)) * (1.0f / cost(tiles[tile].z)) * pieces));
        };
        const int part = (int)blockIdx.x + min(lane, 1), parts = (int)gridDim.x;  // lane 0: where the CTA begins, 1: where it ends
        int tile = 0, in = 0;
        float place = 0.0f;
        if (count > 0) {
            place = (float)(all * part) / parts, tile = tile_at(place, 0, count);
            in = part == 0 ? 0 : part == parts ? p.Ng : piece_at(place, tile, p.Ng);
            place = front(tile) + (float)in / p.Ng * cost(tiles[tile].z);
        }
        const int first_tile = __shfl_sync(0xffffffffu, tile, 0), last_tile = __shfl_sync(0xffffffffu, tile, 1);
        const float from = __shfl_sync(0xffffffffu, place, 0), to = __shfl_sync(0xffffffffu, place, 1);
        const int stripe = tile * p.Ng + in;
        s0 = __shfl_sync(0xffffffffu, stripe, 0), r = __shfl_sync(0xffffffffu, stripe, 1) - s0;
        mine = lane == 0 ? 0 : r * C;
        if (r > 0 && lane > 0 && lane < kWarps) {
            place = from + (to - from) * (lane * (1.0f / kWarps)), tile = tile_at(place, first_tile, last_tile + 1);
            mine = max(0, min(r * C, tile * p.Ng * C + piece_at(place, tile, p.Ng * C) - s0 * C));
        }
    }
    const int begin = __shfl_sync(0xffffffffu, mine, warp), end = __shfl_sync(0xffffffffu, mine, warp + 1);
    WarpRing<G, QTYPE> ring{};
    if (end > begin) {
        uint8_t* slots = smem + p.ring_off + warp * p.depth * S::kSlot;
        const int stripe = begin / C, kc = begin - stripe * C, sg = s0 + stripe, tile = sg / p.Ng, ls = sg - tile * p.Ng;
        ring.slot = slots, ring.at = smem_u32(slots), ring.bar = bars, ring.left = end - begin, ring.tile = tile;
        ring.in_stripe = C - kc, ring.in_tile = (p.Ng - ls) * C - kc;
        ring.from = p.wq + tiles[tile].x * p.group_bytes + ((int64_t)ls * p.Kg + kc * S::kBlocks) * S::BS;
        for (int i = 0; i < p.depth; i++) {
            if (ring.left > 0) ring.ask(p, tiles);
            ring.step(p);
        }
        ring.parity = 0;
    }
    __syncwarp();
    pdl_wait_prior_grid();
    pdl_launch_dependents();

    // four columns of a row to y
    auto store = [&](int64_t n, int place, float4 v) {
        float* y = p.y + (int64_t)__ldcg(p.order + place) * p.ldy + n;
        if (p.y_vec && n + 4 <= p.N) {
            *reinterpret_cast<float4*>(y) = v;
        } else {
            if (n < p.N) y[0] = v.x;
            if (n + 1 < p.N) y[1] = v.y;
            if (n + 2 < p.N) y[2] = v.z;
            if (n + 3 < p.N) y[3] = v.w;
        }
    };
#pragma unroll 1
    for (int c = begin; c < end;) {
        const int li = c / C, kc0 = c - li * C, kc1 = min(C, kc0 + end - c);
        c += kc1 - kc0;
        const int sg = s0 + li, ti = sg / p.Ng;
        const int4 tile = tiles[ti];
        const int64_t n = (int64_t)(sg - ti * p.Ng) * 32 + 4 * g;
        const bool whole = kc0 == 0 && kc1 == C;
        // a row of the tile, all of the stripe or this warp's part of it
        auto put = [&](int row, float4 v) {
            if (row >= tile.z) return;
            if (whole) store(n, tile.y + row, v);
            else *reinterpret_cast<float4*>(part(warp, c == end) + row * 32 + 4 * g) = v;
        };
        // rows row, row + 1 of this lane's four columns
        auto put_two = [&](int row, const uint64_t (&acc)[4]) {
            const float2 v[4] = {unpair(acc[0]), unpair(acc[1]), unpair(acc[2]), unpair(acc[3])};
            put(row, make_float4(v[0].x, v[1].x, v[2].x, v[3].x));
            put(row + 1, make_float4(v[0].y, v[1].y, v[2].y, v[3].y));
        };
        uint64_t acc[2][4];
        uint64_t(&one)[1][4] = reinterpret_cast<uint64_t(&)[1][4]>(acc);
        if (tile.z <= 4) {
            const bool two = tile.z <= 2;
            if (two) walk<G, QTYPE, SIGNED, 4, 1>(p, tiles, ring, fail, lane, tile, ti, kc0, kc1, one);
            else walk<G, QTYPE, SIGNED, 2, 1>(p, tiles, ring, fail, lane, tile, ti, kc0, kc1, one);
#pragma unroll
            for (int k = 0; k < 4; k++) {  // the K groups of the other lanes
                acc[0][k] = add2(acc[0][k], __shfl_xor_sync(0xffffffffu, acc[0][k], 2));
                const uint64_t o = __shfl_xor_sync(0xffffffffu, acc[0][k], 1);
                if (two) acc[0][k] = add2(acc[0][k], o);
            }
            if (t < (two ? 1 : 2)) put_two(2 * t, acc[0]);
        } else if (tile.z <= 8) {
            walk<G, QTYPE, SIGNED, 1, 1>(p, tiles, ring, fail, lane, tile, ti, kc0, kc1, one);
            put_two(2 * t, acc[0]);
        } else {
            walk<G, QTYPE, SIGNED, 1, 2>(p, tiles, ring, fail, lane, tile, ti, kc0, kc1, acc);
            put_two(2 * t, acc[0]);
            put_two(8 + 2 * t, acc[1]);
        }
    }
    // Stripes that several warps have walked, a warp each; lane w knows what warp w has walked.  (Lane i asks for row i of a stripe's tile
    // ahead: row by row, each in its turn, these loads took 6 us with 16 rows.)
    auto rows_of = [&](int li) {
        if (li >= r) return 0;
        const int4 tile = tiles[(s0 + li) / p.Ng];
        return lane < tile.z ? __ldcg(p.order + tile.y + lane) : 0;
    };
    int next = rows_of(warp);
    __syncthreads();
    const int first = mine, after = __shfl_down_sync(0xffffffffu, mine, 1), last = lane < kWarps ? after : first;
    for (int li = warp; li < r; li += kWarps) {
        const int at = next;
        next = rows_of(li + kWarps);
        const bool part_of = first < last && first < (li + 1) * C && last > li * C;
        const uint32_t who = __ballot_sync(0xffffffffu, part_of), ends = __ballot_sync(0xffffffffu, part_of && last <= (li + 1) * C);
        if ((who & (who - 1)) == 0) continue;
        const int sg = s0 + li, ti = sg / p.Ng;
        const int4 tile = tiles[ti];
        const int64_t n = (int64_t)(sg - ti * p.Ng) * 32 + lane;
        for (int row0 = 0; row0 < tile.z; row0 += 4) {
            float sum[4] = {};
            for (uint32_t left = who; left; left &= left - 1) {
                const int w = __ffs(left) - 1;
                const float* from = part(w, ends >> w & 1) + row0 * 32 + lane;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (row0 + k < tile.z) sum[k] += from[k * 32];
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float* y = p.y + (int64_t)__shfl_sync(0xffffffffu, at, row0 + k) * p.ldy + n;
                if (row0 + k < tile.z && n < p.N) *y = sum[k];
            }
        }
    }
    if (*fail != 0) {
        // a wait ran out: copies that may still be in flight land before the shared memory is handed to another CTA
        for (int i = 0; i < 64; i++) __nanosleep(32000);
    }
}

template <int G, int QTYPE, bool SIGNED>
int launch_few(FewParams p, const DeviceInfo* di, cudaStream_t s) {
    using S = FewShape<G, QTYPE>;
    static std::atomic<bool> attr_done[64] = {};  // set once per device; a second setter repeats the same call
    auto* fn = experts_few_kernel<G, QTYPE, SIGNED>;
    if (di->index >= 64 || !attr_done[di->index]) {
        Q4FC_CUDA_OK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, di->max_smem_optin));
        if (di->index < 64) attr_done[di->index] = true;
    }
    p.part_off = (int)align_up(kWarps * kMaxDepth * 8 + 16 + kWarps * 4 + (size_t)p.most_tiles * 16, 128);
    p.ring_off = p.part_off + kWarps * p.part_rows * 128;
    // What the rings leave of the SM's memory is L1, and codes and scales come through it: 64 experts x 1408 x 2048, group
    // 32, with rings of 2 and 3 chunks a warp 16 rows each 42.6 and 43.6 us (of 4, before, 3 more), one row 27.2 and 27.1.
    p.depth = p.weigh ? 2 : kMaxDepth;
    DependentLaunch l(dim3((unsigned)di->sm_count), kThreads, s);
    l.cfg.dynamicSmemBytes = (size_t)p.ring_off + (size_t)p.depth * kWarps * S::kSlot;
    Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, fn, p));
    return Q4FC_OK;
}

}  // namespace

// Up to 96 rows an expert in the mean with group 32, up to 20 with group 128, whose 64-row tiles on tcgen05 have a quarter of the groups to
// scale.  This kernel and those tiles, us, whole call, 32 experts x 2048 x 2048: group 32, 16 rows 38 and 72, 64 rows 105 and 142, 96
// rows 165 and 193; group 128, 16 rows 33 and 39, 20 rows 39 and 40, 32 rows 53 and 44; 8 x 4096 x 8192: group 32, 64 rows 219 and 272, 96
// rows 301 and 348; group 128, 20 rows 64 and 65, 24 rows 71 and 65.  (Its list of stripes is counted in 32 bits.)
bool experts_few_serves(int64_t rows, int64_t Kg, int64_t Ng, int G, int64_t n) {
    const int64_t tiles = most_tiles(kTiles16, rows, n);
    return rows <= (G == 32 ? 96 : 20) * n && tiles <= kMostTiles && (Kg * G + 127) / 128 * Ng * tiles <= 0x7fffffffLL / 8;
}

size_t experts_few_scratch(int64_t rows, int64_t Kg, int G, int64_t n) {
    const int64_t chunks = (Kg * G + 127) / 128;
    return align_up((size_t)(rows * chunks) * 128, 256) + align_up((size_t)(most_tiles(kTiles16, rows, n) * chunks * (128 / G)) * 128, 256);
}

int launch_experts_few(const ExpertsCall& c, GroupQuant q, cudaStream_t s) {
    const DeviceInfo* di = device_info();
    if (!di) return Q4FC_ECUDA;
    const int64_t chunks = (c.Kg * c.G + 127) / 128, tiles = most_tiles(kTiles16, c.rows, c.n);
    const bool sgn = (c.flags & Q4FC_FLAG_NIBBLE_SIGNED) && c.qtype == 0;
    FewParams p = {};
    p.status = ring_status_word();
    if (!p.status) return Q4FC_ECUDA;
    q.codes = reinterpret_cast<int8_t*>(c.scratch), q.sc = reinterpret_cast<float*>(c.scratch + align_up((size_t)(c.rows * chunks) * 128, 256));
    q.tile0 = c.plan.tile0[kTiles16], q.log2tile = 4, q.sums = 1, q.isum = sgn;
    if (int rc = launch_quant_x_group(q, c.G, false, s)) return rc;
    p.codes = q.codes, p.sc = q.sc, p.wq = c.wq, p.y = c.y, p.N = c.N, p.ldy = c.ldy;
    p.tiles = c.plan.tiles[kTiles16], p.tile_count = c.plan.counts + kTiles16, p.order = c.plan.order;
    p.row_bytes = chunks * 128, p.group_bytes = c.Ng * c.Kg * block_bytes(c.qtype, c.G);
    p.Ng = (int)c.Ng, p.Kg = (int)c.Kg, p.chunks = (int)chunks, p.most_tiles = (int)tiles, p.part_rows = (int)(c.most_rows < kTileRows ? c.most_rows : kTileRows);
    p.last_bytes = (int)(c.Kg - (chunks - 1) * (128 / c.G)) * block_bytes(c.qtype, c.G);
    // (beyond two rows the arithmetic takes longer than the bytes)
    p.weigh = c.most_rows > 2;
    p.y_vec = c.ldy % 4 == 0 && (reinterpret_cast<uintptr_t>(c.y) & 15) == 0;
    if (c.qtype == 1) return c.G == 32 ? launch_few<32, 1, false>(p, di, s) : launch_few<128, 1, false>(p, di, s);
    if (!sgn) return c.G == 32 ? launch_few<32, 0, false>(p, di, s) : launch_few<128, 0, false>(p, di, s);
    return c.G == 32 ? launch_few<32, 0, true>(p, di, s) : launch_few<128, 0, true>(p, di, s);
}

}  // namespace q4fc
