// Pre-quantized activations of the decode FC (rows <= 8), by the warp: what quant_x_pre_kernel (quant_x.cu) and the adapters'
// launch in front of a decode FC (lora.cu) share.
#pragma once
#include "common.cuh"

namespace q4fc {

__device__ __forceinline__ int sat8(int v) { return min(127, max(-128, v)); }

// Quantizer in front of the decode FC when rows x K is large.  The decode kernel normally quantizes the
// activations itself, every cluster for itself; from 16K values (quantizes_in_front in fc_decode_ring_impl.cuh)
// that repeated work costs more than one extra small launch.  One warp owns 128 consecutive k of ONE row, so the whole input is
// spread over hundreds of warps and the kernel is a single short latency chain.  Codes and scales follow
// the same rules as quant_x_kernel; the group sums are formed in exactly the order of the decode kernel's
// own quantizer (four values per lane in k order, then a butterfly over the group's lanes), so the FC
// result does not depend on which of the two quantized the input.
//   codes: int8 [rows][Kg*G];   sc: fp32 [Kg][16], entry 2*m = scale d of row m, entry 2*m + 1 = group sum
//   (or, for the signed-nibble Q4_0 form, the bits of the integer 8 * sum of codes).
//
// With `up` given the value that is quantized is silu(x) * up -- the MLP's gate activation and the product with
// the up projection (llmops.itrans(gate, "silu") then llmops.imul(up, gate), ops/op_misc.hpp:83-138,
// chatllama/main.py:365-368), i.e. the input of the down projection -- and `prod`, when given, receives those
// fp32 values.  silu(g) = g / (1 + exp(-g)) with expf and an IEEE division; the reference evaluates exp by a
// degree-5 polynomial and the reciprocal by _mm256_rcp_ps (relative error up to 3.7e-4), so the products agree
// with it to about 4e-4 relative, inside the 1e-3 / 1e-4 output tolerance, not bit for bit.
template <int G>
__device__ __forceinline__ void quant_pre_unit(const float* __restrict__ x, int rows, int64_t K, int64_t ldx, int64_t Kg,
                                               int vec_ok, int want_isum, int early_release, int8_t* __restrict__ codes,
                                               float* __restrict__ sc, const float* __restrict__ up,
                                               float* __restrict__ prod, int64_t ldp, int64_t unit) {
    constexpr int SEG = G / 4;
    constexpr int GPC = 128 / G;
    const int lane = threadIdx.x & 31;
    const int64_t chunks = (Kg * G + 127) / 128;
    // In a chain of programmatic launches the FC kernel behind this one should start as early as it can:
    // its start-up then runs beside the FC before.
    if (early_release) pdl_launch_dependents();
    if (unit >= chunks * rows) return;  // (an exited warp counts as having released the dependent launch)
    const int64_t c = unit / rows;
    const int m = (int)(unit - c * rows);
    const int64_t k = c * 128 + lane * 4;
    const int64_t kb = c * GPC + lane / SEG;
    const bool exists = kb < Kg;
    const int len = exists ? (int)min((int64_t)G, K - kb * G) : 0;
    const int body = len & ~7;
    const int e0 = (lane % SEG) * 4;
    pdl_wait_prior_grid();  // the activations may come from the kernel before

    float v[4] = {0.f, 0.f, 0.f, 0.f};
    const float* src = x + m * ldx + k;
    if (vec_ok && k + 4 <= K) {
        const float4 a = __ldcg(reinterpret_cast<const float4*>(src));
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (k + j < K) v[j] = __ldcg(src + j);
    }
    if (up != nullptr) {
        float u[4] = {0.f, 0.f, 0.f, 0.f};
        const float* usrc = up + m * ldx + k;
        if (vec_ok && k + 4 <= K) {
            const float4 a = __ldcg(reinterpret_cast<const float4*>(usrc));
            u[0] = a.x, u[1] = a.y, u[2] = a.z, u[3] = a.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (k + j < K) u[j] = __ldcg(usrc + j);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float sg = __fdiv_rn(v[j], __fadd_rn(1.0f, expf(-v[j])));
            v[j] = __fmul_rn(u[j], sg);
        }
        if (prod != nullptr) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (k + j < K) prod[m * ldp + k + j] = v[j];
        }
    }
    float amax = 0.0f, fsum = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (e0 + j < len) {
            amax = fmaxf(amax, fabsf(v[j]));
            fsum += v[j];
        }
    // Otherwise the FC kernel behind this launch is released only now, with this warp's activations in
    // registers: its first act is to request megabytes of weights, and these few loads would queue behind
    // that stream.
    if (!early_release) pdl_launch_dependents();
#pragma unroll
    for (int off = SEG / 2; off > 0; off >>= 1) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        fsum += __shfl_xor_sync(0xffffffffu, fsum, off);
    }
    const float d = div_const_rn(amax, 127.0f, 1.0f / 127.0f);
    const float id = inv_or_zero(d);
    uint32_t packed = 0;
    int isum = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        int q = 0;
        if (e0 + j < len) {
            const float t = __fmul_rn(v[j], id);
            if (e0 + j < body) {
                q = __float2int_rn(t);
            } else {
                q = round_half_away(t);  // std::round
            }
            q = sat8(q);
        }
        isum += q;
        packed |= (uint32_t)(q & 0xFF) << (8 * j);
    }
    if (want_isum) {
#pragma unroll
        for (int off = SEG / 2; off > 0; off >>= 1) isum += __shfl_xor_sync(0xffffffffu, isum, off);
    }
    if (exists) {
        *reinterpret_cast<uint32_t*>(codes + m * (Kg * G) + k) = packed;
        if (e0 == 0) {
            sc[kb * 16 + m * 2 + 0] = d;
            sc[kb * 16 + m * 2 + 1] = want_isum ? __int_as_float(8 * isum) : fsum;
        }
    }
}

// The same as a part of another launch: blocks from `first_block` of its grid on.
struct QuantPre {
    const float* x;
    int rows;
    int64_t K, ldx;
    int G, want_isum;
    int8_t* codes;
    float* sc;
    int first_block;
    int64_t units() const { return G ? ((K + G - 1) / G * G + 127) / 128 * rows : 0; }
};
__device__ __forceinline__ void quant_pre_block(const QuantPre& q, int64_t unit) {
    const int vec_ok = q.K % 4 == 0 && q.ldx % 4 == 0 && (reinterpret_cast<uintptr_t>(q.x) & 15) == 0;
    if (q.G == 32) quant_pre_unit<32>(q.x, q.rows, q.K, q.ldx, (q.K + 31) / 32, vec_ok, q.want_isum, 0, q.codes, q.sc, nullptr, nullptr, 0, unit);
    else quant_pre_unit<128>(q.x, q.rows, q.K, q.ldx, (q.K + 127) / 128, vec_ok, q.want_isum, 0, q.codes, q.sc, nullptr, nullptr, 0, unit);
}

}  // namespace q4fc
