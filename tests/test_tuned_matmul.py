"""Which calls of ops.tuned_matmul share one choice of BLAS library.  The timing is stood in for, so no GPU is needed."""
import pytest
import torch

from dms_amd import ops


@pytest.fixture
def timed(monkeypatch):
    """The (rows, type) of every timing round; hipBLASLt is the faster one for 16 bits, rocBLAS for 32."""
    rounds, used = [], []

    def time_matmul(name, a, b):
        if name == "cublas":
            rounds.append((a.shape[0], a.dtype))
        return float((name == "cublas") == (a.dtype != torch.float32))

    monkeypatch.setattr(ops, "_BMM_CHOICE", {})
    monkeypatch.setattr(ops, "_time_matmul", time_matmul)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.backends.cuda, "preferred_blas_library", lambda name=None: used.append(name) or "cublas")
    monkeypatch.delenv("DMN_GEMM_TUNE", raising=False)
    return rounds, used


def test_each_type_has_a_choice_of_its_own(timed):
    rounds, used = timed
    x, w = torch.ones(4, 8), torch.ones(8, 3)
    for dtype, want in ((torch.float32, "cublas"), (torch.bfloat16, "cublaslt"), (torch.float16, "cublaslt"), (torch.float32, "cublas")):
        y = ops.tuned_matmul(x.to(dtype), w.to(dtype))
        assert y.dtype == dtype and used[-2] == want           # the last call puts back what was preferred before
    assert rounds == [(4, torch.float32), (4, torch.bfloat16), (4, torch.float16)]


def test_lengths_between_two_powers_of_two_share_one(timed):
    rounds, _ = timed
    w = torch.ones(8, 3)
    for rows in (40, 33, 64, 50, 65, 128, 1, 2, 100):
        assert ops.tuned_matmul(torch.ones(rows, 8), w, any_rows=True).shape == (rows, 3)
    assert [r for r, _ in rounds] == [40, 65, 1, 2] and len(ops._BMM_CHOICE) == 4
    ops.tuned_matmul(torch.ones(64, 8), w)                     # a shape of its own
    ops.tuned_matmul(torch.ones(63, 8), w)
    assert [r for r, _ in rounds][4:] == [64, 63]


def test_layer_does_not_time_every_length(timed):
    import dms_amd
    rounds, _ = timed
    layer = dms_amd.LinearAttention(8, 16, 2)
    with torch.no_grad():
        for rows in range(33, 65):
            layer._product(torch.ones(rows, 8), layer.weight)
            layer._product(torch.ones(rows, 8), layer.gate)
    assert len(rounds) == 2
