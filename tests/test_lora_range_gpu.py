"""The adapters' projection in half precision over the type's range, against 64 bits.

What lies between the two products (x A^T, dy B) is not of the inputs' type and may be far
smaller or larger than a half-precision number holds well: gradients early in fine-tuning,
large scales.  Tolerances, elementwise and from the data (u = 2^-11, v = 2^-24, tiny =
2^-24, the least subnormal, which only the outputs' own rounding may cost):
  t = dy B     fp32 sums of N products, then two parts of the type, scaled by a power of two
               common to 16 rows of the adapter whose largest lies above 2^6 then:
               |dt| <= N v (|dy| |B|) + 2^-21 |t| + 2^-31 max_adapter |t|
  dA           a sum over the R rows of the adapter:
               |ddA| <= u |dA| + tiny + c (|dt| + (R + 4) v |t|)^T |x|
  dx           the shared product may be rounded before the adapters' part is added, or take
               c t rounded to the type into its sum, in rows whose largest c |t| the type holds
               to full precision (half a step of it for each of the row):
               |ddx| <= 2 (u |dx| + tiny) + u |dy W| + N v (|dy| |W|)
                        + c (|dt| + (r + 4) v |t| + u max_row |t|) |A|
  y, dB        the same with s = x A^T, K for N, dy for x and B for A.
"""
import pytest
import torch

import moe_overlap_b200 as mo
from tests.test_lora_gpu import V, assert_close, make

pytestmark = pytest.mark.gpu

U, TINY = 2.0 ** -11, 2.0 ** -24


def low(x, a):
    """x a^T in 64 bits, how far its two parts and the shared product's operand may be off."""
    s = x @ a.t()
    top = s.abs().max() if s.numel() else 0.0
    ds = x.shape[1] * V * (x.abs() @ a.abs().t()) + 2.0 ** -21 * s.abs() + 2.0 ** -31 * top
    row = s.abs().amax(dim=1, keepdim=True) if s.numel() else s.abs()
    return s, ds, ds + (a.shape[0] + 4) * V * s.abs() + U * row


def reference(x, w, a, b, dy, scale, ids):
    x, w, a, b, dy, scale = (t.detach().double() for t in (x, w, a, b, dy, scale))
    K, N = x.shape[1], w.shape[0]
    y, dx = x @ w.t(), dy @ w
    ty, tx = U * y.abs() + K * V * (x.abs() @ w.abs().t()), U * dx.abs() + N * V * (dy.abs() @ w.abs())
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    ta, tb = torch.zeros_like(a), torch.zeros_like(b)
    for i in range(a.shape[0]):
        rows = (ids == i).nonzero()[:, 0]
        c, R = float(scale[i]), rows.numel()
        if R == 0:
            continue
        s, ds, es = low(x[rows], a[i])
        t, dt, et = low(dy[rows], b[i].t())
        y[rows] += c * (s @ b[i].t())
        ty[rows] += abs(c) * (es @ b[i].abs().t())
        dx[rows] += c * (t @ a[i])
        tx[rows] += abs(c) * (et @ a[i].abs())
        da[i] = c * (t.t() @ x[rows])
        ta[i] = abs(c) * ((dt + (R + 4) * V * t.abs()).t() @ x[rows].abs())
        db[i] = c * (dy[rows].t() @ s)
        tb[i] = abs(c) * (dy[rows].abs().t() @ (ds + (R + 4) * V * s.abs()))
    return ((y, ty + 2 * (U * y.abs() + TINY)), (dx, tx + 2 * (U * dx.abs() + TINY)),
            (da, ta + U * da.abs() + TINY), (db, tb + U * db.abs() + TINY))


def check(x, w, a, b, dy, scale, ids):
    for t in (x, a, b):
        t.requires_grad_(True)
    y = mo.lora_linear(x, w, a, b, ids, scale=scale)
    grads = torch.autograd.grad(y, (x, a, b), dy, retain_graph=True)
    mo.check_status(x.device, sync=True)
    want = reference(x, w, a, b, dy, scale, ids)
    for name, got, ref in zip(("y", "dx", "da", "db"), (y, *grads), want):
        assert bool((ref[0].abs() < 65504).all()), name  # the case stays in the outputs' range
        assert_close(got, ref)
    with torch.no_grad():  # the kernels for few rows, where the batch takes them
        assert_close(mo.lora_linear(x, w, a, b, ids, scale=scale), want[0])
    for one, two in zip(torch.autograd.grad(y, (x, a, b), dy), grads):
        assert torch.equal(one, two)


SIZES = [(40, 264, 328, 3, 8), (512, 256, 1024, 4, 8), (700, 520, 264, 3, 64), (600, 136, 264, 20, 24),
         (300, 1040, 264, 5, 128), (1500, 136, 136, 2, 40)]


@pytest.mark.parametrize("M,K,N,L,r", SIZES)
@pytest.mark.parametrize("std", [1e-3, 1e-4, 1e-5, 1e-6])
def test_small_gradients(cuda_device, M, K, N, L, r, std):
    """dA is a sum over rows, which lifts it out of the subnormal numbers that dy B is among."""
    x, w, a, b, dy, scale, ids = make(M, K, N, L, r, torch.float16, seed=M + r, device=cuda_device)
    check(x, w, a, b, (dy.float() * (10 * std)).half(), scale, ids)


@pytest.mark.parametrize("M,K,N,L,r", SIZES)
def test_small_gradients_and_a_small_second_matrix(cuda_device, M, K, N, L, r):
    x, w, a, b, dy, scale, ids = make(M, K, N, L, r, torch.float16, seed=M + N, device=cuda_device)
    check(x * 16, w, a, (b.float() * 1e-2).half(), (dy.float() * 1e-3).half(), scale * 8, ids)


@pytest.mark.parametrize("M,K,N,L,r", SIZES)
def test_large_low_rank_products(cuda_device, M, K, N, L, r):
    """c x A^T of some rows beyond the type's largest number, their outputs within it."""
    x, w, a, b, dy, scale, ids = make(M, K, N, L, r, torch.float16, seed=M + K, device=cuda_device)
    x[::5] *= 100
    scale = scale * 4096
    check(x, w, (a.float() * 4).half(), (b.float() * 2e-4).half(), dy * 0.01, scale, ids)


@pytest.mark.parametrize("M,K,N,L,r", SIZES)
def test_rows_of_every_size(cuda_device, M, K, N, L, r):
    """Rows over eight orders of magnitude in every adapter, zeros among them."""
    x, w, a, b, dy, scale, ids = make(M, K, N, L, r, torch.float16, seed=M * 3, device=cuda_device)
    g = torch.Generator().manual_seed(r)
    by = 10.0 ** (torch.rand(M, 1, generator=g) * 6 - 5)
    by[::11] = 0
    x = (x.float() * by.to(cuda_device)).half()
    by = 10.0 ** (torch.rand(M, 1, generator=g) * 6 - 5)
    by[3::13] = 0
    check(x, w, a, b, (dy.float() * by.to(cuda_device)).half(), scale, ids)
