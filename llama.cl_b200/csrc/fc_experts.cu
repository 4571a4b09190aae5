// FC by expert: the product of the (token, slot) pairs of a plan (groups.cuh) with the weights that the router chose.  No
// counterpart in the reference; per pair the arithmetic is that of fc_Q4A (ops/op_fc.hpp:286-426).
//
//   h[t, s] = quantized(x[t]) . W[ids[t, s]]            and with weights  y[t] = sum_s weight[t, s] * h[t, s]
//
// Launches: the quantizer, which writes the pairs' codes in the plan's order (quant_x.cu), one kernel for all experts, and
// with weights the sum over the slots, in their order, in fp32 (a token's pairs lie in different experts' tiles).
#include "groups.cuh"

namespace q4fc {
namespace {

struct Combine {
    const float *h, *weights;  // [tokens * top_k][ldh]
    float* y;
    int64_t tokens, N, ldh, ldy;
    unsigned per;  // CTAs of a token
    int top_k;
};
// V columns a thread.  Bound by h and y at many tokens: 4096 of them, 8 slots, 4096 columns, 604 MB in 96 us; 2048, 2 slots, 22016, 541 MB in 118.
template <int V>
__global__ void __launch_bounds__(256) combine_kernel(const Combine a) {
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    const int64_t t = blockIdx.x / a.per, n = ((int64_t)(blockIdx.x % a.per) * 256 + threadIdx.x) * V;
    if (n >= a.N) return;
    float sum[V] = {};
#pragma unroll 4
    for (int s = 0; s < a.top_k; s++) {
        const float w = __ldcg(a.weights + t * a.top_k + s);
        const float* h = a.h + (t * a.top_k + s) * a.ldh + n;
        if constexpr (V == 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(h));
            sum[0] = fmaf(w, v.x, sum[0]), sum[1] = fmaf(w, v.y, sum[1]), sum[2] = fmaf(w, v.z, sum[2]), sum[3] = fmaf(w, v.w, sum[3]);
        } else {
            sum[0] = fmaf(w, __ldcg(h), sum[0]);
        }
    }
    float* y = a.y + t * a.ldy + n;
    if constexpr (V == 4)
        *reinterpret_cast<float4*>(y) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    else
        *y = sum[0];
}

int launch_combine(Combine c, cudaStream_t s) {
    const bool vec = c.N % 4 == 0 && c.ldy % 4 == 0 && (reinterpret_cast<uintptr_t>(c.y) & 15) == 0;
    const int64_t per = (c.N + (vec ? 1023 : 255)) / (vec ? 1024 : 256), grid = c.tokens * per;
    if (grid > 0x7fffffffLL) {
        set_error("fc_experts: %lld tokens x %lld exceeds the grid limit", (long long)c.tokens, (long long)c.N);
        return Q4FC_ELIMIT;
    }
    c.per = (unsigned)per;
    DependentLaunch l(dim3((unsigned)grid), 256, s);
    Q4FC_CUDA_OK(cudaLaunchKernelEx(&l.cfg, vec ? combine_kernel<4> : combine_kernel<1>, c));
    return Q4FC_OK;
}

size_t hidden_bytes(int64_t rows, int64_t N, bool weighted) { return weighted ? align_up((size_t)(rows * N) * 4, 256) : 0; }

}  // namespace

size_t experts_scratch_bytes(int64_t rows, int64_t K, int64_t N, int G, int64_t n, bool weighted) {
    const int64_t Kg = (K + G - 1) / G;
    // (what serves a call depends on its packed tensor's columns too, which may be more than N)
    const size_t gemm = experts_gemm_scratch(rows, Kg, G, n), few = experts_few_serves(rows, Kg, 1, G, n) ? experts_few_scratch(rows, Kg, G, n) : 0;
    return hidden_bytes(rows, N, weighted) + (few > gemm ? few : gemm);
}

int launch_fc_experts(ExpertsCall c, const float* weights, int64_t top_k, cudaStream_t s) {
    const Combine sum = {reinterpret_cast<const float*>(c.scratch), weights, c.y, c.rows / top_k, c.N, c.N, c.ldy, 0, (int)top_k};
    if (weights) {
        c.y = reinterpret_cast<float*>(c.scratch), c.ldy = c.N;
        c.scratch += hidden_bytes(c.rows, c.N, true);
    }
    GroupQuant q = {};
    q.x = c.x, q.rows = c.rows, q.K = c.K, q.Kg = c.Kg, q.ldx = c.ldx, q.per_row = c.per_row, q.gated = c.gated;
    q.group_of = c.plan.group_of, q.place_of = c.plan.place_of, q.offsets = c.plan.offsets, q.n = (int)c.n;
    q.vec_ok = c.K % 4 == 0 && c.ldx % 4 == 0 && (reinterpret_cast<uintptr_t>(c.x) & 15) == 0;
    q.y = c.y, q.N = c.N, q.ldy = c.ldy;
    if (int rc = experts_few_serves(c.rows, c.Kg, c.Ng, c.G, c.n) ? launch_experts_few(c, q, s) : launch_experts_gemm(c, q, s)) return rc;
    return weights ? launch_combine(sum, s) : Q4FC_OK;
}

}  // namespace q4fc
