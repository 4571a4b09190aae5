// FC by expert for few rows: the decode kernel (fc_decode_ring_impl.cuh, EXPERTS = true) over the plan's tiles of up to eight
// rows.  Which experts have rows is known on the device alone, so the launch is one CTA per SM whatever the plan says, and
// every CTA cuts its share out of (tiles in use) x stripes itself; a weight stripe is read once for up to eight rows.
#include "fc_decode_ring_impl.cuh"

#include "groups.cuh"

namespace q4fc {
namespace {

constexpr int64_t kMostPairs = 128;  // what a CTA keeps of the plan: 4 KB

template <int G, int QTYPE, bool SIGNED>
RingVariant* variant_for(int rows) {
    return rows <= 1 ? ring_variant_of<G, QTYPE, SIGNED, 1, false, true, true>() : ring_variant_of<G, QTYPE, SIGNED, 8, false, true, true>();
}
RingVariant* variant_of(int qtype, int G, bool sgn, int rows) {
    if (qtype == 1) return G == 32 ? variant_for<32, 1, false>(rows) : variant_for<128, 1, false>(rows);
    if (!sgn) return G == 32 ? variant_for<32, 0, false>(rows) : variant_for<128, 0, false>(rows);
    return G == 32 ? variant_for<32, 0, true>(rows) : variant_for<128, 0, true>(rows);
}

struct RingFit {
    int cs, nc, kc_max, code_stride, inbox_stripes, part_off, depth;
    size_t fixed;
};
// The shape of the launch; false where the shared memory does not hold it.
bool ring_fit(const ExpertsCall& c, int rows_max, RingVariant* v, const DeviceInfo* di, int dev, RingFit* f) {
    const int64_t tiles = most_tiles(kTiles8, c.rows, c.n), stripes = tiles * c.Ng;
    const int Kg = (int)c.Kg, rows_p = (rows_max + 1) / 2 * 2, slot_bytes = kRW * (c.G == 32 ? 4 : 1) * block_bytes(c.qtype, c.G);
    f->part_off = (int)align_up(512 + (size_t)tiles * 16 + (size_t)c.rows * 4, 128);
    int cs = 1;
    while (cs < 8 && cs * 2 <= Kg && stripes * cs * 2 <= di->sm_count) cs *= 2;
    for (;; cs *= 2) {
        int log2cs = 0;
        while ((1 << log2cs) < cs) log2cs++;
        f->cs = cs, f->kc_max = (Kg + cs - 1) / cs;
        f->code_stride = (f->kc_max * c.G + 127) / 128 * 128 + 32;  // rows 32 B apart modulo 128: conflict-free operand loads
        int cap = di->sm_count / cs;
        if (cs > 1 && (cap = ring_max_clusters(v, dev, cs, log2cs, di)) < 0) return false;
        f->nc = cap < kMaxUnits ? cap : kMaxUnits;
        const int64_t each = (stripes + f->nc - 1) / f->nc;
        f->inbox_stripes = cs > 1 ? (int)((each + cs - 1) / cs) : 0;
        const size_t slot_f = (size_t)rows_p * 32;
        f->fixed = align_up(f->part_off + kPartBufs * kRW * slot_f * 4 + (size_t)f->inbox_stripes * cs * slot_f * 4 + (size_t)f->kc_max * 64 +
                                (size_t)rows_max * f->code_stride, 128);
        if (f->fixed + 2 * (size_t)slot_bytes <= (size_t)di->max_smem_optin) break;
        if (cs >= 8 || cs * 2 > Kg) return false;
    }
    int64_t depth = ((int64_t)di->max_smem_optin - (int64_t)f->fixed) / slot_bytes;
    f->depth = (int)(depth < kRingMax ? depth : kRingMax);
    return true;
}

}  // namespace

bool experts_ring_serves(int64_t rows, int64_t n) { return rows <= kMostPairs && rows <= 8 * n; }

size_t experts_ring_scratch(int64_t rows, int64_t Kg, int G, int64_t n) {
    return align_up((size_t)(rows * Kg * G), 256) + align_up((size_t)(most_tiles(kTiles8, rows, n) * Kg) * 64, 256);
}

int launch_experts_ring(const ExpertsCall& c, GroupQuant q, cudaStream_t s, bool* done) {
    *done = false;
    const DeviceInfo* di = device_info();
    if (!di) return Q4FC_ECUDA;
    int dev = 0;
    Q4FC_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || most_tiles(kTiles8, c.rows, c.n) * c.Ng * c.Kg >= 0x7fffffffLL) return Q4FC_OK;
    const bool sgn = (c.flags & Q4FC_FLAG_NIBBLE_SIGNED) && c.qtype == 0;
    const int rows_max = (int)(c.most_rows < 8 ? c.most_rows : 8);
    RingVariant* v = variant_of(c.qtype, c.G, sgn, rows_max);
    RingFit f;
    if (!ring_fit(c, rows_max, v, di, dev, &f)) return Q4FC_OK;
    {
        std::lock_guard<std::mutex> lk(g_setup_mutex);
        if (!v->attr_done[dev]) {
            Q4FC_CUDA_OK(cudaFuncSetAttribute(v->fn, cudaFuncAttributeMaxDynamicSharedMemorySize, di->max_smem_optin));
            v->attr_done[dev] = true;
        }
    }
    RingExpertParams p = {};
    p.status = ring_status_word();
    if (!p.status) return Q4FC_ECUDA;
    const size_t codes = align_up((size_t)(c.rows * c.Kg * c.G), 256);
    q.codes = reinterpret_cast<int8_t*>(c.scratch), q.sc = reinterpret_cast<float*>(c.scratch + codes);
    q.tile0 = c.plan.tile0[kTiles8], q.log2tile = 3, q.sums = 1, q.isum = sgn;
    if (int rc = launch_quant_x_group(q, c.G, false, s)) return rc;
    p.njobs = p.ninputs = 1;
    p.job[0].wq = c.wq, p.job[0].y = c.y, p.job[0].N = c.N, p.job[0].ldy = c.ldy;
    p.in[0] = {q.codes, q.sc, c.Kg * c.G, c.K, rows_max, (int)c.Kg};
    p.rows_max = rows_max, p.rows_p = (rows_max + 1) / 2 * 2;
    p.cs = f.cs, p.nc = f.nc, p.bq = 1;
    while ((1 << p.log2cs) < f.cs) p.log2cs++;
    p.kq = (int)c.Kg / f.cs, p.kr = (int)c.Kg % f.cs, p.kc_max = f.kc_max, p.code_stride = f.code_stride;
    p.depth = f.depth, p.slot_bytes = kRW * (c.G == 32 ? 4 : 1) * block_bytes(c.qtype, c.G), p.ring_off = (int)f.fixed;
    p.inbox_stripes = f.inbox_stripes;
    p.weights_early = 1;  // (behind the quantizer)
    p.tiles = c.plan.tiles[kTiles8], p.tile_count = c.plan.counts + kTiles8, p.order = c.plan.order;
    p.group_bytes = c.Ng * c.Kg * block_bytes(c.qtype, c.G);
    p.Ng = (int)c.Ng, p.most_tiles = (int)most_tiles(kTiles8, c.rows, c.n), p.pairs = (int)c.rows, p.part_off = f.part_off;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    ring_fill_launch_config(cfg, attr, p.nc * p.cs, p.cs, f.fixed + (size_t)p.depth * p.slot_bytes, true, s);
    void* args[] = {&p};
    Q4FC_CUDA_OK(cudaLaunchKernelExC(&cfg, v->fn, args));
    *done = true;
    return Q4FC_OK;
}

}  // namespace q4fc
