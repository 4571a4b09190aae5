"""Rows sorted by id, and the router: against numpy and against the formula in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg(lib_built):
    assert torch.cuda.is_available()
    import llama_cl_b200

    return llama_cl_b200


def check_plan(groups, ids, n):
    flat = ids.reshape(-1).astype(np.int64)
    key = np.where((flat < 0) | (flat >= n), n, flat)
    order = np.argsort(key, kind="stable")
    offsets = np.searchsorted(key[order], np.arange(n + 1))
    assert np.array_equal(groups.order.cpu().numpy(), order)
    assert np.array_equal(groups.offsets.cpu().numpy(), offsets)
    # the tiles, as the kernels read them
    words = groups.buf.cpu().numpy()
    at = 16 + (n + 4) // 4 * 4 + (flat.size + 3) // 4 * 4
    for i, size in enumerate((8, 16, 64, 128)):
        want = [(g, offsets[g] + k, min(size, offsets[g + 1] - offsets[g] - k), 0)
                for g in range(n) for k in range(0, offsets[g + 1] - offsets[g], size)]
        assert words[i] == len(want)
        assert np.array_equal(words[at: at + 4 * len(want)].reshape(-1, 4), np.array(want, np.int64).reshape(-1, 4))
        at += 4 * (flat.size // size + min(n, flat.size))
    for want in (key, np.argsort(order)):  # the group and the place of each row
        assert np.array_equal(words[at: at + flat.size], want)
        at += (flat.size + 3) // 4 * 4
    for size in (8, 16, 64, 128):
        assert np.array_equal(words[at: at + n + 1], np.cumsum(np.append(0, -(-np.diff(offsets) // size))))
        at += (n + 4) // 4 * 4
    assert at == words.size and not words[4:16].any()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows,n", [(0, 1), (0, 7), (1, 1), (1, 1024), (2, 8), (31, 3), (32, 32), (33, 5), (1023, 2), (1024, 1024),
                                    (2048, 64), (2049, 64), (8192, 1), (8193, 1000), (32768, 128), (262145, 1024)])
def test_group_rows(pkg, rows, n, dtype):
    rng = np.random.default_rng(rows * 1031 + n)
    for low in (0, -n // 2 - 1):  # without and with rows that have no group
        ids = rng.integers(low, n, rows)
        groups = pkg.llmops.group_rows(torch.from_numpy(ids).cuda().to(dtype), n)
        check_plan(groups, ids, n)
    pkg.llmops.check_device_status()


@pytest.mark.parametrize("rows", [5, 5000])
def test_group_rows_of_one_id_and_of_none(pkg, rows):
    for value in (3, -1, -(1 << 31)):
        ids = np.full(rows, value)
        check_plan(pkg.llmops.group_rows(torch.from_numpy(ids).cuda(), 6), ids, 6)
    ids = np.arange(rows)[::-1] % 6
    check_plan(pkg.llmops.group_rows(torch.from_numpy(ids.copy()).cuda().int(), 6), ids, 6)


@pytest.mark.parametrize("bad", [4, 1 << 40])
def test_an_id_beyond_the_last_group_is_reported(pkg, bad):
    ids = np.array([0, bad, 2, -1, 3])
    groups = pkg.llmops.group_rows(torch.from_numpy(ids).cuda(), 4)
    check_plan(groups, ids, 4)
    with pytest.raises(RuntimeError):
        pkg.llmops.check_device_status()
    pkg.llmops.check_device_status()  # read and cleared


def route_64(logits, k, renormalize):
    x = logits.double().cpu().numpy()
    E = x.shape[-1]
    rows = x.reshape(-1, E)
    ids, w = np.full((len(rows), k), -1), np.zeros((len(rows), k))
    for r, row in enumerate(rows):
        open_ = np.nonzero(row > -np.inf)[0]  # (a NaN is not)
        if np.isnan(row).any():
            w[r] = np.nan
        if not len(open_):
            continue
        best = sorted(open_, key=lambda e: (-row[e], e))[:k]
        ids[r, : len(best)] = best
        if not np.isnan(row).any():
            p = np.exp(row - row[open_].max())
            w[r, : len(best)] = p[best] / (p[best].sum() if renormalize else p.sum())
    return ids.reshape(*x.shape[:-1], k), w.reshape(*x.shape[:-1], k)


def check_route(pkg, logits, k, renormalize):
    weights, groups = pkg.llmops.route_top_k(logits, k, renormalize=renormalize)
    ids, want = route_64(logits, k, renormalize)
    assert groups.ids.dtype == torch.int32 and groups.ids.shape == weights.shape == (*logits.shape[:-1], k)
    assert np.array_equal(groups.ids.cpu().numpy(), ids)
    got = weights.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    # a weight is exp(d) / sum: the difference d of two logits is rounded once (2^-24 |d|), expf is off by two units in the last
    # place at most (2^-22), each of up to E additions rounds once and so does the division; |d| is at most 110 where
    # exp(d) is not zero in fp32 (below 2^-126 it is held as a multiple of 2^-149)
    E = logits.shape[-1]
    spread = 110.0
    rel = 2 * (spread * 2.0 ** -24 + 2.0 ** -22) + (E + 1) * 2.0 ** -24
    assert (np.abs(got - want)[fine] <= rel * want[fine] + 2.0 ** -148).all()
    check_plan(groups, ids, E)


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,experts,k", [(0, 4, 2), (1, 1, 1), (1, 8, 2), (3, 32, 32), (7, 33, 5), (64, 64, 6), (65, 100, 8),
                                              (300, 129, 8), (1000, 256, 4), (1025, 1024, 32), (4096, 128, 8)])
def test_route_top_k(pkg, tokens, experts, k, renormalize):
    g = torch.Generator().manual_seed(tokens + experts)
    logits = torch.randn(tokens, experts, generator=g) * 3
    check_route(pkg, logits.cuda(), k, renormalize)


@pytest.mark.parametrize("tokens", [5, 2000])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_equal_closed_and_odd_logits(pkg, tokens, renormalize):
    g = torch.Generator().manual_seed(tokens)
    logits = torch.randint(-2, 3, (1, tokens, 40), generator=g).float()  # many ties
    logits[logits == 0] *= torch.where(torch.rand(int((logits == 0).sum()), generator=g) < 0.5, 1.0, -1.0)  # 0 and -0 are equal
    logits[torch.rand(1, tokens, 40, generator=g) < 0.9] = -float("inf")  # often fewer than top_k are open
    logits[0, 0] = -float("inf")
    logits[0, 1] = torch.finfo(torch.float32).min  # lowest values are open: all equal
    logits[0, 2, 7] = float("nan")
    logits[0, 3] = float("nan")
    logits[0, 4] = 1e30 * torch.arange(40)
    check_route(pkg, logits.cuda(), 6, renormalize)


def test_route_infinite_logit(pkg):
    """exp(inf - inf) is no number, here as in the formula; the choice is made all the same."""
    logits = torch.zeros(2, 4)
    logits[0, 2] = float("inf")
    weights, groups = pkg.llmops.route_top_k(logits.cuda(), 2)
    assert groups.ids.tolist() == [[2, 0], [0, 1]]
    assert weights[0].isnan().any() and weights[1].tolist() == [0.5, 0.5]


def test_route_in_a_graph_and_on_a_stream(pkg):
    """A captured plan follows the inputs of each replay."""
    logits = torch.empty(37, 24, device="cuda")
    first = torch.randn(37, 24, generator=torch.Generator().manual_seed(1)).cuda()
    logits.copy_(first)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        pkg.llmops.route_top_k(logits, 3)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        weights, groups = pkg.llmops.route_top_k(logits, 3)
    for seed in (1, 2):
        logits.copy_(torch.randn(37, 24, generator=torch.Generator().manual_seed(seed)).cuda())
        graph.replay()
        ids, want = route_64(logits, 3, True)
        assert np.array_equal(groups.ids.cpu().numpy(), ids)
        check_plan(groups, ids, 24)


def test_refusals(pkg):
    ops = pkg.llmops
    logits = torch.zeros(2, 4, device="cuda")
    for bad, text in ((lambda: ops.route_top_k(logits, 0), "top_k=0"), (lambda: ops.route_top_k(logits, 5), "top_k=5"),
                      (lambda: ops.route_top_k(logits.half(), 1), "float32"), (lambda: ops.route_top_k(logits[0], 1), "rank 1"),
                      (lambda: ops.route_top_k(logits.t(), 1), "contiguous"), (lambda: ops.route_top_k(logits.cpu(), 1), "CUDA"),
                      (lambda: ops.route_top_k(torch.zeros(1, 64, device="cuda"), 33), "top_k=33"),
                      (lambda: ops.route_top_k(torch.zeros(1, 1025, device="cuda"), 1), "1024 groups"),
                      (lambda: ops.group_rows(logits, 3), "int32 or int64"), (lambda: ops.group_rows(logits.int().t(), 3), "contiguous"),
                      (lambda: ops.group_rows(logits.int().cpu(), 3), "CUDA"), (lambda: ops.group_rows(logits.int(), 0), "1024 groups"),
                      (lambda: ops.group_rows(logits.int(), 1025), "1024 groups")):
        with pytest.raises(RuntimeError, match=text):
            bad()
