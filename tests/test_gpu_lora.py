"""Adapters beside a shared projection against 64 bits: every type and rank, odd sizes, rows without an adapter."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def pkg(lib_built):
    assert torch.cuda.is_available()
    import llama_cl_b200

    return llama_cl_b200


def inputs(rows, n, r, K, N, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + rows * 7 + r)
    x = torch.randn(1, rows, K, generator=g)
    a = (torch.randn(n, r, K, generator=g) / K ** 0.5).to(dtype)
    b = (torch.randn(n, N, r, generator=g) * 0.05).to(dtype)
    return x.cuda(), a.cuda(), b.cuda(), (torch.rand(n, generator=g) + 0.5).cuda()


def added64(x, a, b, scales, ids):
    """What is added to each row in 64 bits, and a bound of the kernel's error.

    An operand of an MMA is cut to 11 bits and its rest to 11 more: a product of fp32 numbers is off by less than 2^-20 of
    it (both rests' roundings and the product of the rests).  An MMA adds eight products to its sum with at most one unit in the last
    place (2^-23) per addition, cut off or rounded: 2^-20 of the absolute terms; a chain has 3 MMAs (hi hi, hi lo, lo hi) for
    eight of its terms, of which two are of rests, 2^-11 of it in size.  Partial sums of warps and slices add at most 24 more roundings."""
    x, a, b = (v.double().cpu().numpy() for v in (x[0], a, b))
    s = np.ones(len(a)) if scales is None else scales.double().cpu().numpy()
    K, r = a.shape[2], a.shape[1]
    want, bound = np.zeros((len(x), b.shape[1])), np.zeros((len(x), b.shape[1]))
    for i in np.unique(ids[ids >= 0]):
        m = ids == i
        t, size = x[m] @ a[i].T, np.abs(x[m]) @ np.abs(a[i]).T
        off = size * ((K // 8 + 4) * 2.0 ** -20 * 1.01 + 24 * 2.0 ** -24 + 2.0 ** -20) + np.abs(t) * 2.0 ** -23
        want[m] = s[i] * (t @ b[i].T)
        bound[m] = s[i] * (off @ np.abs(b[i]).T + (np.abs(t) @ np.abs(b[i]).T) * ((r // 8 + 3) * 2.0 ** -20 * 1.01 + 2.0 ** -20))
    return want, bound + 1e-30


def check(got, want, bound):
    off = np.abs(got.double().cpu().numpy().reshape(want.shape) - want)
    assert (off <= bound).all(), (off / bound).max()


def groups_of(pkg, ids, n):
    return pkg.llmops.group_rows(torch.from_numpy(ids).int().cuda()[None], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,r,K,N", [
    (1, 1, 1, 1, 1), (1, 4, 16, 16, 128), (2, 2, 4, 24, 33), (8, 8, 16, 512, 256), (8, 3, 8, 1000, 130), (9, 2, 12, 77, 100), (40, 70, 64, 264, 96),
    (61, 5, 65, 320, 129), (130, 2, 33, 100, 255), (256, 3, 32, 512, 200), (300, 7, 256, 96, 40), (700, 1, 100, 63, 17), (257, 400, 5, 129, 31)])
def test_lora_add(pkg, rows, n, r, K, N, dtype):
    x, a, b, scales = inputs(rows, n, r, K, N, dtype)
    ids = np.random.default_rng(rows).integers(-1, n, rows)
    if rows == 1:
        ids[:] = n - 1
    groups = groups_of(pkg, ids, n)
    for s in (scales, None):
        want, bound = added64(x, a, b, s, ids)
        y = torch.zeros(1, rows, N, device="cuda")
        pkg.llmops.lora_add(y, x, a, b, groups, scales=s)
        check(y, want, bound)
        # on top of what is there, one rounding more; rows without an adapter are left as they are
        base = torch.randn(1, rows, N, generator=torch.Generator().manual_seed(1)).cuda()
        y = base.clone()
        pkg.llmops.lora_add(y, x, a, b, groups, scales=s)
        there = base[0].double().cpu().numpy()
        check(y, there + want, bound + (np.abs(there) + np.abs(want)) * 2.0 ** -23)
        none = torch.from_numpy(ids < 0).cuda()
        assert torch.equal(y[0, none], base[0, none])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [4, 300])
def test_products_keep_22_bits(pkg, rows, dtype):
    """One term a product: what a single tf32 operand would lose (2^-11) is not lost."""
    n, K, N = 2, 8, 16
    x, a, b, _ = inputs(rows, n, 1, K, N, dtype)
    a[:, :, 1:] = 0
    ids = np.arange(rows) % n
    y = torch.zeros(1, rows, N, device="cuda")
    pkg.llmops.lora_add(y, x, a, b, groups_of(pkg, ids, n))
    want, _ = added64(x, a, b, None, ids)
    # two products, each off by 2^-20 at most (see added64), nothing that cancels
    assert (np.abs(y[0].double().cpu().numpy() - want) <= 2.0 ** -18 * np.abs(want) + 1e-30).all()


@pytest.mark.parametrize("qtype,G", [("q4_0", 32), ("q4_1", 128)])
@pytest.mark.parametrize("rows,K,N", [(1, 512, 96), (8, 4096, 300), (9, 260, 130), (61, 512, 257), (300, 384, 100)])
def test_fc_lora_is_the_two_calls(pkg, rows, K, N, qtype, G):
    ops = pkg.llmops
    n = 3
    x, a, b, scales = inputs(rows, n, 16, K, N, torch.bfloat16)
    wq = ops.offline_FC_quant_Q4A((torch.randn(N, K, generator=torch.Generator().manual_seed(1)) * 0.02).cuda(), qtype=qtype, group_k=G)
    groups = groups_of(pkg, np.arange(rows) % (n + 1) - 1, n)
    for signed in (False, True):
        want = ops.fc_Q4A(x, wq, N, nibble_signed=signed)
        ops.lora_add(want, x, a, b, groups, scales=scales)
        out = torch.full_like(want, float("nan"))
        got = ops.fc_Q4A_lora(x, wq, N, a, b, groups, scales=scales, nibble_signed=signed, out=out)
        assert got is out and torch.equal(got, want)
    ops.check_device_status()


@pytest.mark.parametrize("rows", [5, 280])
def test_views_that_start_anywhere(pkg, rows):
    """Contiguous tensors that start on no 16-byte boundary."""
    n, r, K, N = 2, 16, 64, 64
    x, a, b, scales = inputs(rows, n, r, K, N, torch.float16)
    ids = np.arange(rows) % n
    want, bound = added64(x, a, b, scales, ids)

    def moved(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        v = buf[1:].view(t.shape)
        v.copy_(t)
        return v

    groups = groups_of(pkg, ids, n)
    for which in range(4):
        args = [moved(t) if i == which else t for i, t in enumerate((torch.zeros(1, rows, N, device="cuda"), x, a, b))]
        pkg.llmops.lora_add(*args, groups, scales=scales)
        check(args[0], want, bound)


@pytest.mark.parametrize("rows", [6, 300])
def test_infinities_and_nan_stay_in_their_row(pkg, rows):
    n, r, K, N = 2, 8, 40, 24
    x, a, b, _ = inputs(rows, n, r, K, N, torch.bfloat16)
    groups = groups_of(pkg, np.arange(rows) % n, n)
    y = torch.zeros(1, rows, N, device="cuda")
    pkg.llmops.lora_add(y, x, a, b, groups)
    x[0, 1, 3], x[0, 4, 0] = float("inf"), float("nan")
    again = torch.zeros(1, rows, N, device="cuda")
    pkg.llmops.lora_add(again, x, a, b, groups)
    others = torch.ones(rows, dtype=torch.bool)
    others[[1, 4]] = False
    assert torch.equal(again[0, others], y[0, others]) and again[0, 4].isnan().all() and not again[0, 1].isfinite().any()


@pytest.mark.parametrize("rows", [3, 300])
def test_captured_and_on_two_streams(pkg, rows):
    """Two graphs captured on one stream and replayed on two do not share scratch; a replay follows its inputs."""
    ops = pkg.llmops
    n, K, N = 3, 4096, 256
    x, a, b, scales = inputs(rows, n, 16, K, N, torch.bfloat16)
    wq = ops.offline_FC_quant_Q4A((torch.randn(N, K) * 0.02).cuda())
    ids = torch.zeros(1, rows, dtype=torch.int32, device="cuda")
    xs = [x, torch.randn_like(x)]

    def step(x):
        return ops.fc_Q4A_lora(x, wq, N, a, b, ops.group_rows(ids, n), scales=scales)

    step(x)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in xs], []
    for graph, v in zip(graphs, xs):
        with torch.cuda.graph(graph):
            outs.append(step(v))
    streams = [torch.cuda.Stream() for _ in xs]
    for seed in (1, 2):
        ids.copy_(torch.randint(-1, n, (1, rows), generator=torch.Generator().manual_seed(seed)).int())
        want = [step(v) for v in xs]
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for y, w in zip(outs, want))


def test_empty_sizes(pkg):
    ops = pkg.llmops
    a, b = torch.zeros(2, 4, 32, device="cuda"), torch.zeros(2, 0, 4, device="cuda")
    x = torch.zeros(1, 3, 32, device="cuda")
    wq = ops.offline_FC_quant_Q4A(torch.zeros(32, 32, device="cuda"))
    groups = ops.group_rows(torch.zeros(1, 3, dtype=torch.int32, device="cuda"), 2)
    assert ops.fc_Q4A_lora(x, wq, 0, a, b, groups).shape == (1, 3, 0)
    none = ops.group_rows(torch.zeros(1, 0, dtype=torch.int32, device="cuda"), 2)
    assert ops.fc_Q4A_lora(x[:, :0].contiguous(), wq, 32, a, torch.zeros(2, 32, 4, device="cuda"), none).shape == (1, 0, 32)


def test_refusals(pkg):
    ops = pkg.llmops
    x, a, b, scales = inputs(3, 2, 4, 32, 32, torch.float16)
    wq = ops.offline_FC_quant_Q4A(torch.zeros(32, 32, device="cuda"))
    groups = ops.group_rows(torch.zeros(1, 3, dtype=torch.int32, device="cuda"), 2)
    y = torch.zeros(1, 3, 32, device="cuda")
    call, add = ops.fc_Q4A_lora, ops.lora_add
    wide = torch.zeros(2, 257, 32, dtype=torch.half, device="cuda")
    for bad, text in (
            (lambda: call(x.half(), wq, 32, a, b, groups), "float32"), (lambda: call(x[0], wq, 32, a, b, groups), "rank 2"),
            (lambda: call(x, wq, 32, a.double(), b, groups), "lora_a: must be"), (lambda: call(x, wq, 32, a, b.float(), groups), "lora_b"),
            (lambda: call(x, wq, 32, a[..., :16].contiguous(), b, groups), "lora_a: expected"),
            (lambda: call(x, wq, 31, a, b, groups), "lora_b: expected"), (lambda: call(x, wq, 32, a.transpose(1, 2), b, groups), "contiguous"),
            (lambda: call(x, wq, 32, a[:1].contiguous(), b[:1].contiguous(), groups), "2 groups for 1 adapters"),
            (lambda: call(x[:, :2].contiguous(), wq, 32, a, b, groups), "do not fit"),
            (lambda: call(x, wq, 32, a, b, groups, scales=scales[:1]), "scales: expected 2"),
            (lambda: call(x, wq, 32, a, b, groups, scales=scales.cpu()), "CUDA"), (lambda: call(x, wq, 32, a.cpu(), b, groups), "CUDA"),
            (lambda: call(x, wq, 32, wide, wide.transpose(1, 2).contiguous()[:, :32], groups), "257"),
            (lambda: call(x, wq[None], 32, a, b, groups), r"is<int8>\(3\)"), (lambda: call(x, wq, 32, a, b, groups, out=y[0]), "out"),
            (lambda: add(y[0], x, a, b, groups), "output"), (lambda: add(y.half(), x, a, b, groups), "float32"),
            (lambda: add(y[:, :2].contiguous(), x, a, b, groups), "out: expected")):
        with pytest.raises(RuntimeError, match=text):
            bad()


@pytest.mark.parametrize("dtype", TYPES)
def test_ranks_of_several_host_threads(pkg, dtype):
    """Ranks that need different amounts of shared memory of one kernel, called at once, each on a stream of its own."""
    import threading

    n, rows, K, N = 2, 256, 64, 64
    failed, sums = [], {}

    def work(rank):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                x, a, b, _ = inputs(rows, n, rank, K, N, dtype)
                groups = groups_of(pkg, np.arange(rows) % n, n)
                y = torch.zeros(1, rows, N, device="cuda")
                for _ in range(2000):
                    pkg.llmops.lora_add(y, x, a, b, groups)
                one = torch.zeros(1, rows, N, device="cuda")
                pkg.llmops.lora_add(one, x, a, b, groups)
                torch.cuda.current_stream().synchronize()
                sums[rank] = (one.cpu(), x, a, b)
        except Exception as e:  # (a thread's error would go nowhere)
            failed.append((rank, str(e)))

    threads = [threading.Thread(target=work, args=(rank,)) for rank in (160, 256, 144, 224)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for one, x, a, b in sums.values():
        check(one, *added64(x, a, b, None, np.arange(rows) % n))


@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("rows,n,r,K,N,dtype", [
    (1, 1, 16, 4096, 256, torch.bfloat16), (4, 4, 16, 11008, 256, torch.float32), (61, 40, 64, 11008, 256, torch.float16),
    (61, 3, 200, 11008, 128, torch.float32), (133, 3, 12, 1001, 299, torch.float32), (255, 255, 128, 8192, 96, torch.bfloat16),
    (255, 255, 128, 8192, 96, torch.float32), (300, 300, 64, 8192, 96, torch.bfloat16), (300, 2, 256, 512, 256, torch.float16),
    (300, 2, 256, 512, 256, torch.float32), (300, 2, 64, 11008, 256, torch.float32), (1270, 7, 202, 2011, 264, torch.float32),
    (2048, 4, 32, 11008, 512, torch.bfloat16)])
def test_long_sums_are_as_good_as_fp32(pkg, rows, n, r, K, N, dtype, positive):
    """In the 2-norm, in units u = 2^-23 of a number in [1, 2), of which a number is 0.7 in the mean.

    Cut to 11 + 11 of 24 bits an operand loses up to 3 u, 1.4 as a root of the mean of squares: 1.2e-7 of it; there are two such in each
    product (x or its sum, fp32 weights): 2.4e-7.  Two MMAs of first bits cut up to one u of their sum, half of it in the mean, the first one on
    0.7 of the sum: 0.7e-7.  At most 128 additions round by 0.3 u, on partial sums of 0.7 of the last or less: 1.9e-7.  Together, as if all had
    one sign, 5e-7 for each of the two products: 1e-6.  (A warp's whole K as one chain of MMAs is off by several times that.)"""
    g = torch.Generator("cuda").manual_seed(1)
    of = torch.abs if positive else (lambda t: t)
    a = of(torch.randn(n, r, K, device="cuda", generator=g) / K ** 0.5).to(dtype)
    b = of(torch.randn(n, N, r, device="cuda", generator=g)).to(dtype)
    x = of(torch.randn(1, rows, K, device="cuda", generator=g))
    ids = np.arange(rows) % n
    y = torch.zeros(1, rows, N, device="cuda")
    pkg.llmops.lora_add(y, x, a, b, groups_of(pkg, ids, n))
    some = range(min(rows, 3 * n + 60, 400))
    want = torch.stack([(x[0, k].double() @ a[ids[k]].double().T) @ b[ids[k]].double().T for k in some])
    assert ((y[0, : len(want)] - want).norm() / want.norm()).item() <= 1e-6


@pytest.mark.parametrize("rows,n,rank,K,N", [(5, 3, 16, 512, 256), (5, 8, 72, 512, 256), (61, 3, 16, 512, 256), (61, 40, 64, 320, 2048),
                                             (133, 3, 12, 251, 301), (300, 4, 32, 512, 256), (40, 3, 16, 512, 257), (40, 3, 16, 250, 256),
                                             (40, 3, 24, 512, 131), (40, 3, 24, 245, 130), (40, 3, 64, 512, 131), (40, 3, 64, 245, 130)])
def test_all_inputs_are_written_directly_in_front(pkg, rows, n, rank, K, N):
    """x, both products' weights, the plan and y change between calls that nothing waits for: a launch that begins early reads the new ones."""
    ops = pkg.llmops
    sets = [inputs(rows, n, rank, K, N, torch.bfloat16, seed=s) for s in range(4)]
    ids = [torch.from_numpy(np.random.default_rng(s).integers(-1, n, rows)).int().cuda()[None] for s in range(4)]
    wq = ops.offline_FC_quant_Q4A((torch.randn(N, -(-K // 4) * 4, generator=torch.Generator().manual_seed(1)) * 0.02).cuda())
    want = [ops.fc_Q4A_lora(x, wq, N, a, b, ops.group_rows(i, n), scales=s) for (x, a, b, s), i in zip(sets, ids)]
    torch.cuda.synchronize()
    x, a, b, s = (torch.empty_like(t) for t in sets[0])
    i, out = torch.empty_like(ids[0]), [torch.full_like(want[0], float("nan")) for _ in sets]

    def refill(k):
        for to, of in zip((x, a, b, s, i), (*sets[k], ids[k])):
            to.copy_(of)

    for _ in range(20):
        for k in range(4):
            refill(k)
            ops.fc_Q4A_lora(x, wq, N, a, b, ops.group_rows(i, n), scales=s, out=out[k])
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(out, want))
        for o in out:
            o.fill_(float("nan"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,rank,K,N", [
    (1, 2, 65, 512, 96), (1, 2, 256, 260, 130), (8, 5, 72, 512, 256), (8, 5, 65, 300, 67), (8, 3, 256, 384, 64), (3, 70, 20, 260, 15361),
    (8, 300, 16, 512, 16384), (61, 5, 65, 512, 257), (61, 40, 72, 512, 256), (133, 7, 256, 300, 131), (133, 100, 20, 132, 4099), (255, 255, 9, 96, 515)])
def test_fc_lora_of_many_ranks_or_columns_is_the_two_calls(pkg, rows, n, rank, K, N, dtype):
    """Where both products are launches of their own: in front of a decode FC, which finds y of the adapters alone and zeros where a row has
    none, and around the GEMM."""
    ops = pkg.llmops
    x, a, b, scales = inputs(rows, n, rank, K, N, dtype)
    wq = ops.offline_FC_quant_Q4A((torch.randn(N, K, generator=torch.Generator().manual_seed(1)) * 0.02).cuda(), qtype="q4_1", group_k=32)
    ids = np.random.default_rng(rows).integers(-1, n, rows)
    ids[rows // 2] = -1
    for some in (ids, np.full(rows, -1), np.full(rows, n - 1)):
        groups = groups_of(pkg, some, n)
        want = ops.fc_Q4A(x, wq, N)
        ops.lora_add(want, x, a, b, groups, scales=scales)
        out = torch.full_like(want, float("nan"))
        assert torch.equal(ops.fc_Q4A_lora(x, wq, N, a, b, groups, scales=scales, out=out), want)
    ops.check_device_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,r,K,N", [(257, 1024, 20, 200, 48), (300, 257, 64, 264, 40), (1024, 1024, 12, 96, 64), (2000, 700, 33, 65, 31)])
def test_as_many_adapters_as_rows_or_more(pkg, rows, n, r, K, N, dtype):
    """Tiles of 64 rows with one or two in use."""
    x, a, b, scales = inputs(rows, n, r, K, N, dtype)
    ids = np.arange(rows) % n
    ids[5::9] = -1
    want, bound = added64(x, a, b, scales, ids)
    y = torch.zeros(1, rows, N, device="cuda")
    pkg.llmops.lora_add(y, x, a, b, groups_of(pkg, ids, n), scales=scales)
    check(y, want, bound)
