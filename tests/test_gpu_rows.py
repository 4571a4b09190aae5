"""FCs whose weights depend on the row, as a model runs them: a layer of experts and Linears with adapters one behind another, captured,
without waiting in between; leading dimensions of the C entry points; offsets beyond 32 bits."""
import ctypes as C

import numpy as np
import pytest
import torch

from fc64 import EPS, fc64
from test_gpu_experts import check, choose, pack, want64
from test_gpu_lora import added64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg(lib_built):
    assert torch.cuda.is_available()
    import llama_cl_b200

    return llama_cl_b200


def linear(N, K, bias=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    m = torch.nn.Linear(K, N, bias=bias)
    with torch.no_grad():
        m.weight.copy_(torch.randn(N, K, generator=g) * 0.05)
        if bias:
            m.bias.copy_(torch.randn(N, generator=g))
    return m


def moe(pkg, n, hidden, inner, top_k, qtype, G, seed=0):
    experts = [(linear(inner, hidden, seed=seed + 3 * e), linear(inner, hidden, seed=seed + 3 * e + 1), linear(hidden, inner, seed=seed + 3 * e + 2))
               for e in range(n)]
    return pkg.ops.llmop_moe_q4a(experts, top_k, qtype=qtype, group_k=G, device="cuda"), experts


@pytest.mark.parametrize("qname,qtype,G", [("q4_0", 0, 32), ("q4_1", 1, 128)])
@pytest.mark.parametrize("tokens,n,top_k,hidden,inner", [(1, 4, 2, 128, 96), (6, 40, 6, 260, 68), (50, 5, 2, 100, 36), (300, 3, 2, 132, 72)])
def test_layer_of_experts(pkg, tokens, n, top_k, hidden, inner, qname, qtype, G):
    """The router, gate and up, silu and the sum of the down projections, each step against 64 bits of what the step in front left."""
    ops = pkg.llmops
    layer, experts = moe(pkg, n, hidden, inner, top_k, qname, G)
    assert torch.equal(layer.down[-1], ops.offline_FC_quant_Q4A(experts[-1][2].weight.detach().cuda(), qtype=qname, group_k=G))
    g = torch.Generator().manual_seed(tokens)
    x, logits = torch.randn(1, tokens, hidden, generator=g).cuda(), torch.randn(1, tokens, n, generator=g)
    logits[0, tokens // 2, 1:] = float("-inf")  # one token with one expert
    logits = logits.cuda()
    got = layer(x, logits)

    weights, groups = ops.route_top_k(logits, top_k)
    p = torch.softmax(logits[0].double().cpu(), -1)
    w64, order = p.sort(dim=-1, descending=True, stable=True)
    w64, order = w64[:, :top_k], order[:, :top_k].clone()
    order[w64 == 0] = -1
    ids = groups.ids[0].cpu()
    assert torch.equal(ids.long(), order)
    assert torch.allclose(weights[0].double().cpu(), w64 / w64.sum(-1, keepdim=True), rtol=1e-5, atol=0)
    both = ops.fc_Q4A_experts(x, layer.gate_up, 2 * inner, groups)
    check(both, *want64(x[0].cpu().numpy(), ids.numpy(), layer.gate_up.cpu().numpy(), 2 * inner, qtype, G))

    gate, up = (v.reshape(1, -1, inner).contiguous() for v in (both[..., :inner], both[..., inner:]))
    products = torch.empty_like(gate)
    for r in range(0, gate.shape[1], 8):
        part = torch.empty_like(gate[:, r: r + 8])
        ops.silu_mul_quantize(gate[:, r: r + 8].contiguous(), up[:, r: r + 8].contiguous(), G, product=part)
        products[:, r: r + 8] = part
    want, bound = want64(products.view(tokens, top_k, inner).cpu().numpy(), ids.numpy(), layer.down.cpu().numpy(), hidden, qtype, G)
    w = weights[0].double().cpu().numpy()[..., None]
    check(got, (want * w).sum(1), (bound * w).sum(1) + top_k * EPS * (np.abs(want) * w).sum(1) + 1e-30)
    assert torch.equal(got, ops.fc_Q4A_experts(both, layer.down, hidden, groups, weights=weights, silu_mul=True))
    ops.check_device_status()


def test_layer_refusals(pkg):
    with pytest.raises(RuntimeError, match="no experts"):
        pkg.ops.llmop_moe_q4a([], 1)
    with pytest.raises(RuntimeError, match="sizes"):
        pkg.ops.llmop_moe_q4a([(linear(8, 32), linear(8, 32), linear(32, 12))], 1)
    with pytest.raises(RuntimeError, match="bias"):
        pkg.ops.llmop_moe_q4a([(linear(8, 32, bias=True), linear(8, 32), linear(32, 8))], 1)
    layer, _ = moe(pkg, 2, 32, 8, 1, "q4_1", 32)
    with pytest.raises(RuntimeError, match="logits of 3"):
        layer(torch.zeros(1, 1, 32, device="cuda"), torch.zeros(1, 1, 3, device="cuda"))
    assert "experts" not in repr(layer) and layer.weight_size() == layer.gate_up.numel() + layer.down.numel()
    a, b = torch.zeros(4, 32), torch.zeros(16, 4)
    with pytest.raises(RuntimeError, match="no adapters"):
        pkg.ops.llmop_fc_q4a_lora(linear(16, 32), [])
    for bad in ((a, b[:8], 1.0), (a[:, :16], b, 1.0), (a[:2], b, 1.0), (a[0], b, 1.0)):
        with pytest.raises(RuntimeError, match="adapter"):
            pkg.ops.llmop_fc_q4a_lora(linear(16, 32), [(a, b, 1.0), bad])


@pytest.mark.parametrize("rows", [1, 8, 70])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_with_adapters(pkg, rows, bias):
    """Adapters of several ranks, one of them without weight, and rows without any."""
    ops, K, N = pkg.llmops, 200, 90
    g = torch.Generator().manual_seed(rows)
    ranks = [4, 16, 9]
    parts = [(torch.randn(r, K, generator=g) / K ** 0.5, torch.randn(N, r, generator=g), s) for r, s in zip(ranks, (2.0, 0.5, 0.0))]
    m = linear(N, K, bias)
    fc = pkg.ops.llmop_fc_q4a_lora(m, parts, group_k=128, device="cuda")
    assert fc.lora_a.shape == (3, 16, K) and fc.lora_b.shape == (3, N, 16) and fc.lora_a.dtype == torch.float32
    x = torch.randn(1, rows, K, generator=g).cuda()
    ids = (np.arange(rows) + 1) % 4 - 1
    got = fc(x, ops.group_rows(torch.from_numpy(ids).cuda()[None], 3))
    want, bound = added64(x, fc.lora_a, fc.lora_b, fc.scales, ids)
    y, off = fc64(x[0].cpu().numpy(), fc.weight.cpu().numpy(), N, 1, 128)
    shift = m.bias.detach().double().numpy() if bias else 0.0
    check(got, y + want + shift, off + bound + (np.abs(y) + np.abs(want) + np.abs(shift)) * 2 * 2.0 ** -23)


@pytest.mark.parametrize("rows", [3, 60])
def test_decoding_steps_in_a_graph(pkg, rows):
    """Projections with adapters, their sum with others, a router on what they leave, the experts: one graph, replayed with other inputs,
    gives the bits of the calls one by one."""
    ops, K, n = pkg.llmops, 256, 6
    g = torch.Generator().manual_seed(rows)
    adapters = [(torch.randn(8, K, generator=g) / 16, torch.randn(K, 8, generator=g) / 4, 1.5) for _ in range(3)]
    first = pkg.ops.llmop_fc_q4a_lora(linear(K, K, seed=9), adapters, dtype=torch.bfloat16, device="cuda")
    wq = ops.offline_FC_quant_Q4A(linear(K, K, seed=10).weight.detach().cuda())
    layer, _ = moe(pkg, n, K, 96, 2, "q4_1", 32)
    router = (torch.randn(n, K, generator=g) / 16).cuda()
    x, ids = torch.empty(1, rows, K, device="cuda"), torch.empty(1, rows, dtype=torch.int32, device="cuda")

    def step():
        groups = ops.group_rows(ids, 3)
        h = x + first(x, groups)
        v = ops.fc_Q4A(h, wq, K)
        ops.lora_add(v, h, first.lora_a, first.lora_b, groups, scales=first.scales)
        h = h + v
        return h + layer(h, (h[..., None, :] * router).sum(-1))

    def refill(seed):
        gen = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(1, rows, K, generator=gen))
        ids.copy_(torch.randint(-1, 3, (1, rows), generator=gen))

    refill(0)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        refill(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert out.isfinite().all() and torch.equal(out, step())
    ops.check_device_status()


@pytest.mark.parametrize("tokens", [1, 7, 90])
def test_calls_without_a_wait_between_them(pkg, tokens):
    """Plans, products and scratch are dropped and their memory taken again while kernels that read them may still run."""
    ops, n, K, N = pkg.llmops, 5, 512, 160
    wq = pack(pkg, n, N, K, 1, 32, 3)
    g = torch.Generator().manual_seed(tokens)
    a, b = (torch.randn(n, 16, K, generator=g) / 16).half().cuda(), torch.randn(n, N, 16, generator=g).half().cuda()
    xs = [torch.randn(1, tokens, K, generator=g).cuda() for _ in range(12)]
    logits = [torch.randn(1, tokens, n, generator=g).cuda() for _ in xs]

    def run(x, l, wait):
        weights, groups = ops.route_top_k(l, 2)
        wait()
        y = ops.fc_Q4A_experts(x, wq, N, groups, weights=weights)
        wait()
        z = ops.fc_Q4A_lora(x, wq[0], N, a, b, ops.group_rows(groups.ids[..., 0].contiguous(), n))
        wait()
        return y + z

    want = [run(x, l, torch.cuda.synchronize) for x, l in zip(xs, logits)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            got = [run(x, l, lambda: None) for x, l in zip(xs, logits)]
            torch.cuda.synchronize()
            assert all(torch.equal(y, w) for y, w in zip(got, want))


def groups_of(pkg, ids, n):
    return pkg.llmops.group_rows(torch.from_numpy(ids).int().cuda()[None], n)


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("G", [32, 128])
@pytest.mark.parametrize("tokens,n", [(3, 6), (60, 3), (230, 2)])
def test_leading_dimensions_of_experts(pkg, tokens, n, G, weighted):
    """Rows of x and y with space behind them: what lies there is left as it was, and not read."""
    L, top_k, K, N = pkg._cabi.lib(), 2, 130, 70
    ldx, ldy = K + 5, N + 3
    ids = choose(np.random.default_rng(tokens), tokens, n, top_k, none=0.1)
    wq, groups = pack(pkg, n, N, K, 1, G, 0), groups_of(pkg, ids, n)
    x = torch.full((tokens + 1, ldx), float("nan"), device="cuda")
    x[:tokens, :K] = torch.randn(tokens, K, generator=torch.Generator().manual_seed(1)).cuda()
    weights = torch.rand(tokens, top_k, generator=torch.Generator().manual_seed(2)).cuda() if weighted else None
    rows = tokens if weighted else tokens * top_k
    y = torch.full((rows + 2, ldy), 7.0, device="cuda")
    ws = torch.empty(L.q4fc_experts_workspace_bytes(tokens, top_k, K, N, G, n, weighted) + 64, dtype=torch.uint8, device="cuda").fill_(0x5A)
    c = pkg._cabi.ExpertsCall(x=x.data_ptr(), tokens=tokens, top_k=top_k, K=K, ldx=ldx, wq=wq.data_ptr(), experts=n, Ng=wq.shape[1], Kg=wq.shape[2],
                              N=N, qtype=1, group_k=G, groups=groups.buf.data_ptr(), weights=weights.data_ptr() if weighted else None,
                              y=y.data_ptr(), ldy=ldy)
    assert L.q4fc_fc_experts(C.byref(c), ws.data_ptr(), ws.numel() - 64, 0, torch.cuda.current_stream().cuda_stream) == 0, L.q4fc_last_error()
    want, bound = want64(x[:tokens, :K].cpu().numpy(), ids, wq.cpu().numpy(), N, 1, G)
    if weighted:
        w = weights.double().cpu().numpy()[..., None]
        bound = (bound * w).sum(1) + top_k * EPS * (np.abs(want) * w).sum(1) + 1e-30
        want = (want * w).sum(1)
    check(y[:rows, :N].contiguous(), want.reshape(rows, N), bound.reshape(rows, N))
    assert (y[rows:] == 7).all() and (y[:, N:] == 7).all() and (ws[-64:] == 0x5A).all()


@pytest.mark.parametrize("with_fc", [False, True])
@pytest.mark.parametrize("rows,rank,ldx,ldy", [(4, 8, 133, 71), (40, 20, 132, 72), (300, 8, 131, 75), (300, 72, 140, 80)])
def test_leading_dimensions_of_adapters(pkg, rows, rank, ldx, ldy, with_fc):
    L, n, K, N = pkg._cabi.lib(), 3, 128, 70
    g = torch.Generator().manual_seed(rows)
    ids = np.arange(rows) % (n + 1) - 1
    x = torch.full((rows + 1, ldx), float("nan"), device="cuda")
    x[:rows, :K] = torch.randn(rows, K, generator=g).cuda()
    a, b = (torch.randn(n, rank, K, generator=g) / 11).bfloat16().cuda(), torch.randn(n, N, rank, generator=g).bfloat16().cuda()
    y = torch.full((rows + 1, ldy), 7.0, device="cuda")
    y[:rows, :N] = 0
    wq = pkg.llmops.offline_FC_quant_Q4A((torch.randn(N, K, generator=g) * 0.05).cuda())
    groups = groups_of(pkg, ids, n)
    need = L.q4fc_fc_lora_workspace_bytes(rows, rank, K, N, 1, 32) if with_fc else L.q4fc_lora_workspace_bytes(rows, rank)
    ws = torch.empty(need + 64, dtype=torch.uint8, device="cuda").fill_(0x5A)
    c = pkg._cabi.LoraCall(x=x.data_ptr(), rows=rows, K=K, ldx=ldx, lora_a=a.data_ptr(), lora_b=b.data_ptr(), dtype=2, adapters=n, rank=rank, N=N,
                           groups=groups.buf.data_ptr(), y=y.data_ptr(), ldy=ldy)
    stream = torch.cuda.current_stream().cuda_stream
    want, bound = added64(x[None, :rows, :K], a, b, None, ids)
    if with_fc:
        rc = L.q4fc_fc_lora(C.byref(c), wq.data_ptr(), wq.shape[0], wq.shape[1], 1, 32, ws.data_ptr(), need, 0, stream)
        base, off = fc64(x[:rows, :K].cpu().numpy(), wq.cpu().numpy(), N, 1, 32)
        want, bound = want + base, bound + off + (np.abs(base) + np.abs(want)) * 2.0 ** -23
    else:
        rc = L.q4fc_lora_add(C.byref(c), ws.data_ptr(), need, stream)
    assert rc == 0, L.q4fc_last_error()
    check(y[:rows, :N].contiguous(), want, bound)
    assert (y[rows:] == 7).all() and (y[:, N:] == 7).all() and (ws[-64:] == 0x5A).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [5, 100, 300])
@pytest.mark.parametrize("rank", [12, 20, 72])
def test_an_infinite_weight_reaches_its_column_alone(pkg, rank, rows, dtype):
    """Ranks that fill no tile are padded with neighbours of other columns: an infinity there must not meet a zero."""
    n, K, N = 2, 32, 48
    g = torch.Generator().manual_seed(rank)
    x = torch.randn(1, rows, K, generator=g).cuda()
    a, b = (torch.randn(n, rank, K, generator=g) / 6).to(dtype).cuda(), torch.randn(n, N, rank, generator=g).to(dtype).cuda()
    groups = groups_of(pkg, np.arange(rows) % n, n)
    want = torch.zeros(1, rows, N, device="cuda")
    pkg.llmops.lora_add(want, x, a, b, groups)
    b[1, 5], b[1, 47, 0], b[0, 0, rank - 1] = float("nan"), float("inf"), float("-inf")
    got = torch.zeros_like(want)
    pkg.llmops.lora_add(got, x, a, b, groups)
    hit = torch.zeros(rows, N, dtype=torch.bool, device="cuda")
    hit[1::2, 5], hit[1::2, 47], hit[::2, 0] = True, True, True
    assert torch.equal(got[0][~hit], want[0][~hit]) and not got[0][hit].isfinite().any()


@pytest.mark.parametrize("G", [32, 128])
@pytest.mark.parametrize("tokens,n,top_k", [(700, 1000, 1), (2000, 1000, 2), (300, 1024, 32), (60, 1024, 4)])
def test_hundreds_of_experts(pkg, tokens, n, top_k, G):
    """As many tiles as the kernel for few rows lists, more than that, and most experts without a row."""
    K, N = 100, 40
    rng = np.random.default_rng(tokens)
    ids = np.stack([rng.choice(n, top_k, replace=False) for _ in range(tokens)])
    ids[: tokens // 8, 0] = n - 1  # one expert with many
    some = pack(pkg, 7, N, K, 1, G, 3)
    wq = some[torch.arange(n, device="cuda") % 7].contiguous()
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, tokens, K, generator=g)
    got = pkg.llmops.fc_Q4A_experts(x.cuda(), wq, N, groups_of(pkg, ids, n))
    check(got, *want64(x[0].numpy(), ids % 7, some.cpu().numpy(), N, 1, G))


def test_experts_beyond_32_bit_offsets(pkg):
    """5 GB of experts, the last one chosen; then 9.6 GB of outputs."""
    ops, n, K, N = pkg.llmops, 1024, 4096, 2048
    one = ops.offline_FC_quant_Q4A((torch.randn(N, K, generator=torch.Generator().manual_seed(1)) * 0.02).cuda(), group_k=128)
    wq = torch.zeros(n, *one.shape, dtype=torch.int8, device="cuda")
    assert wq.numel() > 1 << 32
    wq[-1] = one
    for tokens in (2, 40):
        x = torch.randn(1, tokens, K, generator=torch.Generator().manual_seed(tokens))
        got = ops.fc_Q4A_experts(x.cuda(), wq, N, groups_of(pkg, np.full((tokens, 1), n - 1), n))
        check(got[..., -32:].contiguous(), *(v[:, None] for v in fc64(x[0].numpy(), one[-1:].cpu().numpy(), 32, 1, 128)))
    del wq
    tokens, K, N = 4000, 64, 600000
    wq = torch.zeros(2, N // 32, K // 32, 640, dtype=torch.int8, device="cuda")
    tail = pack(pkg, 2, 32, K, 1, 32, 5)
    wq[:, -1:] = tail
    x = torch.randn(1, tokens, K, generator=torch.Generator().manual_seed(7))
    ids = (np.arange(tokens) % 2)[:, None]
    got = ops.fc_Q4A_experts(x.cuda(), wq, N, groups_of(pkg, ids, 2))
    assert got.numel() > 1 << 31
    want, bound = want64(x[0].numpy(), ids, tail.cpu().numpy(), 32, 1, 32)
    check(got[..., -32:].contiguous(), want, bound)
    assert not got[..., :64].any()


@pytest.mark.parametrize("rows", [6, 300])
def test_adapters_beyond_32_bit_offsets(pkg, rows):
    """5 GB of each adapter weight, the last adapter used; with many rows they are few columns of many: y is small."""
    n, r, K, N = 1024, 72, 32768, 32768
    a, b = torch.zeros(n, r, K, dtype=torch.half, device="cuda"), torch.zeros(n, N, r, dtype=torch.half, device="cuda")
    assert a.numel() > 1 << 31
    g = torch.Generator().manual_seed(1)
    a[-1] = (torch.randn(r, K, generator=g) / K ** 0.5).half().cuda()
    b[-1, -40:] = torch.randn(40, r, generator=g).half().cuda()
    x = torch.randn(1, rows, K, generator=g).cuda()
    y = torch.zeros(1, rows, N, device="cuda")
    pkg.llmops.lora_add(y, x, a, b, groups_of(pkg, np.full(rows, n - 1), n))
    want, bound = added64(x, a[-1:], b[-1:, -40:], None, np.zeros(rows, np.int64))
    check(y[..., -40:].contiguous(), want, bound)
    assert not y[..., :-40].any()


def test_adapters_of_as_many_rows_as_a_plan_holds(pkg):
    """2^23 rows, few columns."""
    rows, n, K, N = 1 << 23, 3, 8, 4
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(1, rows, K, device="cuda", generator=g)
    a, b = torch.randn(n, 2, K, device="cuda", generator=g), torch.randn(n, N, 2, device="cuda", generator=g)
    ids = torch.randint(-1, n, (1, rows), device="cuda", generator=g, dtype=torch.int32)
    groups = pkg.llmops.group_rows(ids, n)
    y = torch.zeros(1, rows, N, device="cuda")
    pkg.llmops.lora_add(y, x, a, b, groups)
    some = torch.cat([torch.arange(200), torch.randint(0, rows, (200,), generator=torch.Generator().manual_seed(2)), torch.arange(rows - 200, rows)])
    want, bound = added64(x[:, some.cuda()], a, b, None, ids[0, some.cuda()].cpu().numpy())
    check(y[0, some.cuda()], want, bound)
    assert not y[0, ids[0] < 0].any()


@pytest.mark.parametrize("tokens", [2, 70, 300])
def test_calls_of_several_host_threads(pkg, tokens):
    """A step of everything, on a stream of its own for each thread: the bits of one thread alone."""
    import threading

    ops, n, K, N = pkg.llmops, 6, 256, 160
    wq = pack(pkg, n, N, K, 1, 128, 3)
    g = torch.Generator().manual_seed(tokens)
    a, b = (torch.randn(n, 160, K, generator=g) / 16).half().cuda(), torch.randn(n, N, 160, generator=g).half().cuda()
    xs = [torch.randn(1, tokens, K, generator=g).cuda() for _ in range(4)]
    logits = [torch.randn(1, tokens, n, generator=g).cuda() for _ in xs]

    def step(i):
        rank = (8, 160, 40, 136)[i]
        la, lb = a[:, :rank].contiguous(), b[..., :rank].contiguous()
        weights, groups = ops.route_top_k(logits[i], 2)
        y = ops.fc_Q4A_experts(xs[i], wq, N, groups, weights=weights)
        rows = ops.group_rows(groups.ids[..., 0].contiguous(), n)
        y = y + ops.fc_Q4A_lora(xs[i], wq[0], N, la, lb, rows)
        ops.lora_add(y, xs[i], la, lb, rows)
        return y

    want = [step(i) for i in range(4)]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(40):
                    got = step(i)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want[i]):
                    failed.append((i, "other bits"))
        except Exception as e:  # (a thread's error would go nowhere)
            failed.append((i, str(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    ops.check_device_status()


@pytest.mark.parametrize("tokens", [3, 60, 300])
def test_branches_of_a_graph(pkg, tokens):
    """Plans made on a side branch, two branches that read one plan, a copy and a fill directly in front of calls."""
    ops, n, K, N = pkg.llmops, 5, 512, 192
    wq, other = pack(pkg, n, N, K, 1, 32, 3), pack(pkg, n, N, K, 0, 128, 4)
    g = torch.Generator().manual_seed(tokens)
    a, b = (torch.randn(n, 16, K, generator=g) / 16).half().cuda(), torch.randn(n, N, 16, generator=g).half().cuda()
    fresh, x = torch.empty(1, tokens, K, device="cuda"), torch.empty(1, tokens, K, device="cuda")
    logits, ids = torch.empty(1, tokens, n, device="cuda"), torch.empty(1, tokens, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()

    def step(side):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            rows = ops.group_rows(ids, n)
            z = torch.zeros(1, tokens, N, device="cuda")
            ops.lora_add(z, fresh, a, b, rows)
        weights, groups = ops.route_top_k(logits, 2)
        x.copy_(fresh)
        y = ops.fc_Q4A_experts(x, wq, N, groups, weights=weights)
        main.wait_stream(side)
        y = y + ops.fc_Q4A_lora(x, wq[0], N, a, b, rows)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            v = ops.fc_Q4A_experts(x, other, N, groups)
        w = ops.fc_Q4A_experts(x, wq, N, groups)
        main.wait_stream(side)
        return y, z, v, w

    def refill(seed):
        gen = torch.Generator().manual_seed(seed)
        fresh.copy_(torch.randn(1, tokens, K, generator=gen))
        logits.copy_(torch.randn(1, tokens, n, generator=gen))
        ids.copy_(torch.randint(-1, n, (1, tokens), generator=gen))

    refill(0)
    step(torch.cuda.current_stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(side)
    for seed in (1, 2, 3):
        refill(seed)
        for _ in range(4):
            graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(u, v) for u, v in zip(got, step(torch.cuda.current_stream())))
    ops.check_device_status()
