"""GPU parity of the few-token experts at sizes where their work divides unevenly; the
tolerances are those of test_few_tokens_gpu.py."""
import pytest
import torch

import moe_overlap_b200 as mo
from tests.test_few_tokens_gpu import V, assert_close, experts64, make, route64

pytestmark = pytest.mark.gpu


def check(device, T, E, H, F, k, dtype, renorm=True, seed=0):
    x, rw, w1, w2 = make(T, E, H, F, dtype, seed=seed, device=device)
    out, idx, w = mo.moe_few_tokens(x, rw, w1, w2, k, renormalize=renorm)
    mo.check_status(device, sync=True)
    want_i, want_w = route64(x, rw, None, k, renorm)
    assert torch.equal(idx, want_i)
    rel = (E + 16) * 2 * V
    assert bool(((w.double() - want_w).abs() <= rel * want_w + 1e-38).all())
    want, tol = experts64(x, w1, w2, want_i, want_w, dw_rel=rel)
    assert_close(out, want, tol)


@pytest.mark.parametrize("T,E,H,F,k,dtype", [
    (14, 2, 8, 73736, 2, torch.bfloat16), (9, 3, 264, 9224, 1, torch.float16), (16, 4, 136, 16392, 3, torch.bfloat16),
    (1, 1, 264, 73736, 1, torch.bfloat16), (2, 4, 72, 20488, 2, torch.float16), (40, 2, 1032, 12296, 2, torch.bfloat16)])
def test_many_parts_of_ffn(cuda_device, T, E, H, F, k, dtype):
    """Long sums of the down-projection: several parts an item, of widths that leave a
    short last one (and, were the parts not counted by their width, an empty one)."""
    check(cuda_device, T, E, H, F, k, dtype, seed=T)


def test_widths_past_what_an_int_holds_are_refused(cuda_device):
    z = torch.zeros(1, dtype=torch.bfloat16, device=cuda_device)
    idx, w = torch.zeros(1, 1, dtype=torch.int64, device=cuda_device), torch.zeros(1, 1, device=cuda_device)
    for H, F in ((2 ** 30 + 8, 8), (8, 2 ** 30 + 8), (2 ** 32 + 8, 8)):  # (views of one element)
        with pytest.raises(ValueError, match="up to 2\\^30"):
            mo.experts_few_tokens(z.expand(1, H), z.expand(1, F, H), z.expand(1, H, F), idx, w)


@pytest.mark.parametrize("T,E,H", [(128, 256, 8), (128, 3, 8), (1, 256, 16), (77, 9, 24)])
def test_gate_of_few_columns(cuda_device, T, E, H):
    """Logits of a column block or two: the gate's CTAs are done with their products before
    the one that gathers them need have started."""
    for seed in range(3):
        check(cuda_device, T, E, H, 16, min(E, 2), torch.bfloat16, seed=seed)
