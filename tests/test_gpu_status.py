"""The device's status word: ids out of range and waits that ran out, side by side."""
import ctypes as C
import os
import subprocess

import pytest
import torch

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
BAD_EMBEDDING, BAD_GROUP = 0x80, 0x8000


@pytest.fixture(scope="module")
def pkg(lib_built):
    assert torch.cuda.is_available()
    import llama_cl_b200

    return llama_cl_b200


@pytest.fixture(scope="module")
def wait_probe(pkg, tmp_path_factory):
    from llama_cl_b200 import build

    try:
        build.nvcc()
    except RuntimeError as e:
        pytest.skip(str(e))
    so = str(tmp_path_factory.mktemp("probe") / "wait_probe.so")
    subprocess.run([build.nvcc(), *build.NVCC_FLAGS, "-shared", "-cudart", "static", os.path.join(HERE, "wait_probe.cu"), "-o", so,
                    "-Xcompiler", "-fvisibility=default"], check=True)
    fn = C.CDLL(so).wait_probe
    fn.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p]
    return fn


@pytest.mark.parametrize("ids", [0, BAD_EMBEDDING, BAD_GROUP, BAD_EMBEDDING | BAD_GROUP])
def test_a_wait_that_runs_out_is_noted_beside_bad_ids(pkg, wait_probe, ids):
    """An id out of range, not read yet, does not hide that results are incomplete."""
    code = int.from_bytes(b"FXPL", "big")
    ws = pkg.llmops.Workspace(4096, torch.device("cuda"))
    word = ws.buf[:4].view(torch.int32)
    word.fill_(ids)
    failed = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert wait_probe(word.data_ptr(), code, failed.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    assert failed.item() == 1 and word.item() == code | ids
    # the first one's code stays
    assert wait_probe(word.data_ptr(), int.from_bytes(b"PREF", "big"), failed.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    assert word.item() == code | ids
    text = [t for bit, t in ((BAD_EMBEDDING, "an embedding id was out of range"), (BAD_GROUP, "an id of an expert or adapter was out of range"))
            if ids & bit] + ["a bounded wait ran out"]
    with pytest.raises(RuntimeError, match=r"\(" + "; ".join(text) + r"\)"):
        ws.check()
    ws.check()  # cleared


def test_a_bad_id_of_a_plan_is_no_bad_embedding(pkg):
    ops = pkg.llmops
    ops.group_rows(torch.tensor([0, 4], device="cuda"), 4)
    with pytest.raises(RuntimeError, match=r"\(an id of an expert or adapter was out of range\)"):
        ops.check_device_status()
    op = pkg.ops.llmop_embedding_q8c(torch.randn(10, 64, device="cuda"))
    op(torch.tensor([10], device="cuda"))
    ops.group_rows(torch.arange(300, device="cuda"), 4)
    with pytest.raises(RuntimeError, match=r"\(an embedding id was out of range; an id of an expert or adapter was out of range\)"):
        ops.check_device_status()
    ops.check_device_status()
