"""Argument checks of the entry points for rows with weights of their own: they come before any CUDA call."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def cabi(lib_built):
    import llama_cl_b200 as pkg

    return pkg._cabi


EINVAL, EVARIANT, EALIGN, EWORKSPACE, ELIMIT = 1, 2, 3, 4, 7


def test_plans(cabi):
    L = cabi.lib()
    assert L.q4fc_groups_bytes(-1, 4) == L.q4fc_groups_bytes(8, 0) == L.q4fc_groups_bytes(8, 1025) == L.q4fc_groups_bytes((1 << 23) + 1, 4) == 0
    assert 0 < L.q4fc_groups_bytes(0, 1) < L.q4fc_groups_bytes(1 << 23, 1024)
    assert L.q4fc_group_rows(16, 1, -1, 4, 16, None) == EINVAL
    assert L.q4fc_group_rows(16, 1, 4, 0, 16, None) == EINVAL
    assert L.q4fc_group_rows(16, 1, 4, 1025, 16, None) == ELIMIT
    assert L.q4fc_group_rows(16, 1, (1 << 23) + 1, 4, 16, None) == ELIMIT
    assert L.q4fc_group_rows(16, 1, 4, 4, None, None) == EINVAL
    assert L.q4fc_group_rows(16, 1, 4, 4, 8, None) == EALIGN
    assert L.q4fc_group_rows(None, 1, 4, 4, 16, None) == EINVAL
    assert L.q4fc_group_rows(12, 0, 4, 4, 16, None) == EINVAL and b"ids" in L.q4fc_last_error()


def test_router(cabi):
    L = cabi.lib()

    def call(logits=16, tokens=2, experts=8, ld=8, top_k=2, weights=16, ids=16, groups=16):
        return L.q4fc_route_top_k(logits, tokens, experts, ld, top_k, 1, weights, ids, groups, None)

    for bad in (dict(top_k=0), dict(top_k=9), dict(tokens=-1), dict(logits=None), dict(weights=None), dict(ids=None), dict(groups=None), dict(ld=7),
                dict(logits=18), dict(ids=18), dict(experts=0, top_k=1)):
        assert call(**bad) == EINVAL, bad
    for bad in (dict(experts=1025, ld=1025), dict(experts=64, ld=64, top_k=33), dict(tokens=1 << 23), dict(tokens=1 << 62)):
        assert call(**bad) == ELIMIT, bad
    assert call(groups=8) == EALIGN


def experts_call(cabi, ws=256, ws_bytes=1 << 30, **change):
    args = dict(x=16, tokens=3, top_k=2, K=64, ldx=64, x_per_slot=0, silu_mul=0, wq=16, experts=4, Ng=1, Kg=2, N=32, qtype=1, group_k=32, groups=16,
                most_rows=0, weights=None, y=16, ldy=32)
    args.update(change)
    return cabi.lib().q4fc_fc_experts(C.byref(cabi.ExpertsCall(**args)), ws, ws_bytes, 0, None)


def test_experts(cabi):
    L = cabi.lib()
    assert L.q4fc_fc_experts(None, 256, 1 << 30, 0, None) == EINVAL
    for change in (dict(tokens=-1), dict(top_k=0), dict(most_rows=-1), dict(experts=0), dict(groups=None), dict(x=None), dict(wq=None), dict(y=None),
                   dict(K=0), dict(K=65), dict(Kg=3), dict(N=33, ldy=33), dict(N=-1), dict(ldx=63), dict(ldy=31), dict(silu_mul=1), dict(ldx=127, silu_mul=1)):
        assert experts_call(cabi, **change) == EINVAL, change
    for change in (dict(qtype=2), dict(group_k=64)):
        assert experts_call(cabi, **change) == EVARIANT, change
    for change in (dict(top_k=33), dict(tokens=1 << 23), dict(tokens=1 << 40), dict(experts=1025)):
        assert experts_call(cabi, **change) == ELIMIT, change
    for change in (dict(groups=8), dict(wq=8), dict(weights=18), dict(ws=128), dict(x=18)):
        assert experts_call(cabi, **change) == EALIGN, change
    need = L.q4fc_experts_workspace_bytes(3, 2, 64, 32, 32, 4, 0)
    assert need > 0 and experts_call(cabi, ws_bytes=need - 1) == EWORKSPACE and experts_call(cabi, ws=None) == EWORKSPACE
    assert L.q4fc_experts_workspace_bytes(3, 2, 64, 32, 32, 4, 1) > need
    assert experts_call(cabi, tokens=0, x=None, y=None) == 0 and experts_call(cabi, N=0) == 0
    for bad in ((-1, 2, 64, 32, 32, 4), (3, 0, 64, 32, 32, 4), (3, 33, 64, 32, 32, 4), (3, 2, 0, 32, 32, 4), (3, 2, 64, -1, 32, 4), (3, 2, 64, 32, 48, 4),
                (3, 2, 64, 32, 32, 0), (3, 2, 64, 32, 32, 1025), (1 << 23, 2, 64, 32, 32, 4)):
        assert L.q4fc_experts_workspace_bytes(*bad, 0) == 0, bad


def lora_call(cabi, fc=False, ws=256, ws_bytes=1 << 30, flags=0, wq=16, Ng=1, Kg=2, qtype=1, group_k=32, **change):
    args = dict(x=16, rows=3, K=64, ldx=64, lora_a=16, lora_b=16, dtype=2, adapters=4, rank=8, N=32, scales=None, groups=16, y=16, ldy=32)
    args.update(change)
    call = cabi.LoraCall(**args)
    if fc:
        return cabi.lib().q4fc_fc_lora(C.byref(call), wq, Ng, Kg, qtype, group_k, ws, ws_bytes, flags, None)
    return cabi.lib().q4fc_lora_add(C.byref(call), ws, ws_bytes, None)


@pytest.mark.parametrize("fc", [False, True])
def test_adapters(cabi, fc):
    for change in (dict(rows=-1), dict(K=0), dict(N=-1), dict(rank=0), dict(adapters=0), dict(groups=None), dict(x=None), dict(lora_a=None),
                   dict(lora_b=None), dict(y=None), dict(ldx=63), dict(ldy=31), dict(dtype=3)):
        assert lora_call(cabi, fc, **change) == EINVAL, change
    for change in (dict(rank=257), dict(adapters=1025), dict(rows=(1 << 23) + 1), dict(K=1 << 30, ldx=1 << 30)):
        assert lora_call(cabi, fc, **change) == ELIMIT, change
    for change in (dict(groups=8), dict(lora_a=17), dict(lora_b=18, dtype=0), dict(scales=18), dict(y=18), dict(ws=128)):
        assert lora_call(cabi, fc, **change) == EALIGN, change
    assert lora_call(cabi, fc, ws=None) == lora_call(cabi, fc, ws_bytes=64) == EWORKSPACE
    assert lora_call(cabi, fc, rows=0, x=None, y=None) == 0 and lora_call(cabi, fc, N=0) == 0


def test_adapters_beside_an_fc(cabi):
    L = cabi.lib()
    for change in (dict(wq=None), dict(Kg=3), dict(Ng=0), dict(flags=4)):
        assert lora_call(cabi, True, **change) == EINVAL, change
    assert lora_call(cabi, True, group_k=64) == EVARIANT
    assert lora_call(cabi, True, ws_bytes=L.q4fc_lora_workspace_bytes(3, 8)) == EWORKSPACE
    assert L.q4fc_lora_workspace_bytes(3, 257) == L.q4fc_lora_workspace_bytes(-1, 8) == L.q4fc_lora_workspace_bytes(3, 0) == 0
    assert L.q4fc_fc_lora_workspace_bytes(3, 8, 64, 32, 2, 32) == L.q4fc_fc_lora_workspace_bytes(3, 8, 0, 32, 1, 32) == 0
    assert L.q4fc_fc_lora_workspace_bytes(3, 8, 64, 32, 1, 32) > L.q4fc_lora_workspace_bytes(3, 8)


def test_wrappers_reject_cpu_tensors(lib_built):
    import torch

    import llama_cl_b200 as pkg

    ops = pkg.llmops
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.group_rows(torch.zeros(3, dtype=torch.int32), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.route_top_k(torch.zeros(3, 4), 2)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        ops.group_rows(torch.zeros(3), 2)
