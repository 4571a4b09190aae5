"""FC by expert against 64 bits: every block type, rows per token and per pair, sums over the slots, ragged sizes, experts with no
row, one row and many, tokens without an expert."""
import numpy as np
import pytest
import torch

from fc64 import EPS, fc64

pytestmark = pytest.mark.gpu

BLOCKS = [(0, 32), (0, 128), (1, 32), (1, 128)]


@pytest.fixture(scope="module")
def pkg(lib_built):
    assert torch.cuda.is_available()
    import llama_cl_b200

    return llama_cl_b200


def pack(pkg, n, N, K, qtype, G, seed):
    """K need not be a multiple of four, which the packer wants: columns beyond it are zeros."""
    g = torch.Generator().manual_seed(seed)
    w = torch.zeros(n, N, -(-K // 4) * 4)
    w[..., :K] = torch.randn(n, N, K, generator=g) * 0.02
    return torch.stack([pkg.llmops.offline_FC_quant_Q4A(v.cuda(), qtype=qtype, group_k=G) for v in w])


def want64(x, ids, wq, N, qtype, G, signed=False):
    """x fp32 [tokens, K] or [tokens, top_k, K], ids [tokens, top_k] -> products and bounds [tokens, top_k, N]."""
    y, bound = np.zeros((*ids.shape, N)), np.zeros((*ids.shape, N))
    for e in np.unique(ids[ids >= 0]):
        t, s = np.nonzero(ids == e)
        y[t, s], bound[t, s] = fc64(x[t] if x.ndim == 2 else x[t, s], wq[e], N, qtype, G, signed)
    return y, bound


def check(got, want, bound):
    got = got.double().cpu().numpy().reshape(want.shape)
    off = np.abs(got - want)
    assert (off <= bound).all(), f"{(off / np.maximum(bound, 1e-300)).max()} of the bound at {np.argmax(off - bound)}"


def call_and_check(pkg, ids, n, K, N, qtype, G, per_slot=False, weighted=False, seed=0, signed=False, distinct=False):
    tokens, top_k = ids.shape
    g = torch.Generator().manual_seed(seed + 1)
    x = torch.randn(1, tokens, *((top_k,) if per_slot else ()), K, generator=g)
    wq = pack(pkg, n, N, K, qtype, G, seed)
    groups = pkg.llmops.group_rows(torch.from_numpy(ids).int().cuda()[None], n)
    groups.distinct = distinct
    weights = torch.rand(1, tokens, top_k, generator=g) if weighted else None
    want, bound = want64(x[0].numpy(), ids, wq.cpu().numpy(), N, qtype, G, signed)
    out = torch.full((1, tokens, N) if weighted else (1, tokens, top_k, N), float("nan"), device="cuda")
    got = pkg.llmops.fc_Q4A_experts(x.cuda(), wq, N, groups, weights=weights.cuda() if weighted else None, nibble_signed=signed, out=out)
    assert got is out
    if weighted:
        w = weights[0].double().numpy()[..., None]
        bound = (bound * w).sum(1) + top_k * EPS * (np.abs(want) * w).sum(1) + 1e-30  # (a fused addition a slot)
        want = (want * w).sum(1)
    check(got, want, bound)
    pkg.llmops.check_device_status()


def choose(rng, tokens, n, top_k, skew=0.0, none=0.0):
    ids = np.stack([rng.permutation(n)[:top_k] for _ in range(tokens)]) if tokens else np.zeros((0, top_k), np.int64)
    if skew:
        for t in np.nonzero(rng.random(tokens) < skew)[0]:  # most tokens take expert 0
            if 0 not in ids[t]:
                ids[t, 0] = 0
    ids[rng.random(ids.shape) < none] = -1
    return ids


@pytest.mark.parametrize("qtype,G", BLOCKS)
@pytest.mark.parametrize("tokens,n,top_k,K,N", [
    (1, 8, 2, 256, 64), (1, 4, 1, 128, 32), (2, 3, 3, 384, 100), (5, 16, 4, 515, 77), (8, 8, 2, 1000, 33), (9, 2, 2, 250, 130),
    (33, 5, 2, 321, 257), (64, 7, 3, 640, 96), (130, 3, 2, 100, 129), (200, 2, 1, 513, 200), (300, 4, 3, 260, 40)])
def test_products(pkg, tokens, n, top_k, K, N, qtype, G):
    ids = choose(np.random.default_rng(tokens + K), tokens, n, top_k)
    call_and_check(pkg, ids, n, K, N, qtype, G, seed=tokens)
    call_and_check(pkg, ids, n, K, N, qtype, G, seed=tokens, distinct=True)  # a token's experts are different ones


@pytest.mark.parametrize("qtype,G", BLOCKS)
@pytest.mark.parametrize("tokens,n,top_k,K,N", [(1, 8, 2, 512, 96), (3, 6, 4, 300, 35), (17, 9, 5, 129, 64), (150, 2, 2, 384, 131),
                                                (90, 40, 6, 96, 70)])
def test_rows_per_pair_and_sums_over_slots(pkg, tokens, n, top_k, K, N, qtype, G):
    ids = choose(np.random.default_rng(tokens + K), tokens, n, top_k, none=0.1)
    call_and_check(pkg, ids, n, K, N, qtype, G, per_slot=True, weighted=True, seed=tokens)
    call_and_check(pkg, ids, n, K, N, qtype, G, per_slot=False, weighted=True, seed=tokens + 1)
    call_and_check(pkg, ids, n, K, N, qtype, G, per_slot=True, seed=tokens + 2)


@pytest.mark.parametrize("G", [32, 128])
@pytest.mark.parametrize("tokens", [3, 50, 300])
def test_signed_nibbles(pkg, tokens, G):
    ids = choose(np.random.default_rng(tokens), tokens, 4, 2)
    call_and_check(pkg, ids, 4, 328, 90, 0, G, signed=True)


@pytest.mark.parametrize("qtype,G", [(1, 32), (0, 128)])
@pytest.mark.parametrize("tokens,n,top_k", [(1, 3, 2), (7, 12, 2), (40, 64, 4), (257, 64, 4), (700, 6, 2)])
def test_skewed_experts_and_tokens_without_one(pkg, tokens, n, top_k, qtype, G):
    rng = np.random.default_rng(tokens)
    call_and_check(pkg, choose(rng, tokens, n, top_k, skew=0.8, none=0.3), n, 264, 65, qtype, G)
    call_and_check(pkg, np.full((tokens, top_k), -1), n, 264, 65, qtype, G)
    call_and_check(pkg, np.full((tokens, top_k), -1), n, 264, 65, qtype, G, weighted=True)
    ids = np.full((tokens, top_k), -1)
    ids[-1, -1] = n - 1  # one pair in all
    call_and_check(pkg, ids, n, 264, 65, qtype, G)


@pytest.mark.parametrize("tokens", [1, 6, 20, 100])
def test_one_expert_for_all_and_the_same_twice(pkg, tokens):
    """All pairs in one expert, a token's slots among them: more rows than tokens."""
    call_and_check(pkg, np.full((tokens, 3), 1), 3, 200, 70, 1, 32)
    call_and_check(pkg, np.full((tokens, 3), 1), 3, 200, 70, 1, 128, weighted=True)


@pytest.mark.parametrize("qtype,G", BLOCKS)
@pytest.mark.parametrize("tokens,K,N", [(1, 4096, 512), (3, 11008, 96), (12, 2816, 1000), (40, 5000, 40), (150, 4096, 150)])
def test_long_rows(pkg, tokens, K, N, qtype, G):
    """K divided over clusters, and long sums."""
    ids = choose(np.random.default_rng(tokens), tokens, 4, 2)
    call_and_check(pkg, ids, 4, K, N, qtype, G)


@pytest.mark.parametrize("tokens", [1, 4, 8, 30, 128])
@pytest.mark.parametrize("K", [64, 257, 1408])
def test_silu_mul(pkg, tokens, K):
    """What is quantized is what silu_mul_quantize quantizes, bit for bit: its products go through the formula here."""
    ops = pkg.llmops
    g = torch.Generator().manual_seed(tokens + K)
    ids = choose(np.random.default_rng(tokens), tokens, 5, 2, none=0.1)
    rows = torch.randn(1, tokens, 2, 2 * K, generator=g).cuda()
    gate, up = (v.reshape(1, -1, K).contiguous() for v in (rows[..., :K], rows[..., K:]))
    products = torch.empty_like(gate)
    for r in range(0, gate.shape[1], 8):
        part = torch.empty_like(gate[:, r: r + 8])
        ops.silu_mul_quantize(gate[:, r: r + 8].contiguous(), up[:, r: r + 8].contiguous(), 32, product=part)
        products[:, r: r + 8] = part
    wq = pack(pkg, 5, 75, K, 1, 32, 3)
    groups = ops.group_rows(torch.from_numpy(ids).cuda()[None], 5)
    got = ops.fc_Q4A_experts(rows, wq, 75, groups, silu_mul=True)
    check(got, *want64(products.view(tokens, 2, K).cpu().numpy(), ids, wq.cpu().numpy(), 75, 1, 32))


@pytest.mark.parametrize("tokens", [2, 40, 200])
def test_odd_rows(pkg, tokens):
    """Rows of zeros, one large value, values that leave nothing of the others; infinities stay in their own row."""
    rng = np.random.default_rng(tokens)
    ids = choose(rng, tokens, 3, 2)
    x = rng.standard_normal((tokens, 300)).astype(np.float32)
    x[0] = 0
    x[1, 5] = 1e30
    x[tokens // 2, ::7] = 1e-38
    wq = pack(pkg, 3, 64, 300, 1, 32, 1)
    groups = pkg.llmops.group_rows(torch.from_numpy(ids).cuda()[None], 3)
    want, bound = want64(x, ids, wq.cpu().numpy(), 64, 1, 32)
    got = pkg.llmops.fc_Q4A_experts(torch.from_numpy(x).cuda()[None], wq, 64, groups)
    check(got, want, bound)
    x[1, 6] = np.inf
    again = pkg.llmops.fc_Q4A_experts(torch.from_numpy(x).cuda()[None], wq, 64, groups)
    others = np.arange(tokens) != 1
    assert torch.equal(again[0, others], got[0, others])


@pytest.mark.parametrize("tokens,n", [(2, 8), (30, 4), (400, 3)])
def test_captured_and_on_two_streams(pkg, tokens, n):
    """A captured router and product follow the inputs of each replay; two calls at once do not share scratch; the same bits again."""
    ops = pkg.llmops
    g = torch.Generator().manual_seed(tokens)
    wq = pack(pkg, n, 160, 512, 1, 128, 1)
    logits, x = torch.randn(1, tokens, n, generator=g).cuda(), torch.randn(1, tokens, 512, generator=g).cuda()

    def step():
        weights, groups = ops.route_top_k(logits, 2)
        return ops.fc_Q4A_experts(x, wq, 160, groups, weights=weights)

    step()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    streams = [torch.cuda.Stream() for _ in range(2)]
    for seed in (1, 2):
        gen = torch.Generator().manual_seed(seed)
        logits.copy_(torch.randn(1, tokens, n, generator=gen).cuda())
        x.copy_(torch.randn(1, tokens, 512, generator=gen).cuda())
        want = step()
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        eager = []
        for stream in streams:
            with torch.cuda.stream(stream):
                eager.append(step())
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in outs + eager)


@pytest.mark.parametrize("tokens", [0, 3])
def test_empty_sizes(pkg, tokens):
    ops = pkg.llmops
    wq = pack(pkg, 2, 32, 64, 1, 32, 0)
    groups = ops.group_rows(torch.zeros(1, tokens, 2, dtype=torch.int32, device="cuda"), 2)
    x = torch.zeros(1, tokens, 64, device="cuda")
    assert ops.fc_Q4A_experts(x, wq, 0, groups).shape == (1, tokens, 2, 0)
    if tokens == 0:
        assert ops.fc_Q4A_experts(x, wq, 32, groups).shape == (1, 0, 2, 32)
        assert ops.fc_Q4A_experts(x, wq, 32, groups, weights=torch.zeros(1, 0, 2, device="cuda")).shape == (1, 0, 32)


def test_refusals(pkg):
    ops = pkg.llmops
    wq = pack(pkg, 2, 64, 64, 1, 32, 0)
    groups = ops.group_rows(torch.zeros(1, 3, 2, dtype=torch.int32, device="cuda"), 2)
    x = torch.zeros(1, 3, 64, device="cuda")
    call = ops.fc_Q4A_experts
    for bad, text in (
            (lambda: call(x.cpu(), wq, 64, groups), "CUDA"), (lambda: call(x.half(), wq, 64, groups), "float32"),
            (lambda: call(x[0], wq, 64, groups), "rank 2"), (lambda: call(torch.zeros(1, 3, 128, device="cuda")[..., ::2], wq, 64, groups), "contiguous"),
            (lambda: call(x, wq[0], 64, groups), r"is<int8>\(4\)"), (lambda: call(x, wq[:, :1], 32, groups), "contiguous"),
            (lambda: call(x, wq[..., :600].contiguous(), 64, groups), "block size 600"), (lambda: call(x, wq, 65, groups), "65"),
            (lambda: call(x, wq, -1, groups), "negative"), (lambda: call(x[..., :32].contiguous(), wq, 64, groups), "K=32"),
            (lambda: call(x[:, :2].contiguous(), wq, 64, groups), "do not fit"),
            (lambda: call(x[:, :, None].contiguous(), wq, 64, groups), "do not fit"),
            (lambda: call(x, wq[:1].contiguous(), 64, groups), "2 groups for 1 experts"),
            (lambda: call(x, wq, 64, groups, weights=torch.zeros(1, 3, 1, device="cuda")), "weights: expected shape"),
            (lambda: call(x, wq, 64, groups, weights=torch.zeros(1, 3, 2)), "CUDA"),
            (lambda: call(x, wq, 64, groups, out=torch.zeros(1, 3, 64, device="cuda")), "out"),
            (lambda: call(x[..., :63].contiguous(), wq, 64, groups, silu_mul=True), "even"),
            (lambda: call(x, wq, 64, groups, silu_mul=True), "K=32")):
        with pytest.raises(RuntimeError, match=text):
            bad()
    other = ops.group_rows(torch.zeros(1, 3, 2, dtype=torch.int32, device="cuda"), 2)
    other.buf = other.buf[:-4]
    with pytest.raises(RuntimeError, match="not a plan"):
        call(x, wq, 64, other)


@pytest.mark.parametrize("qtype,signed", [(0, False), (0, True), (1, False)])
@pytest.mark.parametrize("K,N", [(11008, 7040), (11008, 4100), (4096, 9000), (1000, 300)])
def test_one_expert_for_64_rows_is_the_fc(pkg, K, N, qtype, signed):
    """The same tiles, K divided as often and long sums moved as often: the same bits."""
    wq = pkg.llmops.offline_FC_quant_Q4A((torch.randn(N, K, generator=torch.Generator().manual_seed(1)) * 0.02).cuda(), qtype=qtype, group_k=128)
    x = torch.randn(1, 64, K, generator=torch.Generator().manual_seed(2)).cuda()
    groups = pkg.llmops.group_rows(torch.zeros(1, 64, 1, dtype=torch.int32, device="cuda"), 1)
    got = pkg.llmops.fc_Q4A_experts(x, wq[None], N, groups, nibble_signed=signed)
    assert torch.equal(got[:, :, 0], pkg.llmops.fc_Q4A(x, wq, N, nibble_signed=signed))
    pkg.llmops.check_device_status()
