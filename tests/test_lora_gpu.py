"""GPU parity of the adapters' projection and its gradients against 64 bits.

Tolerances, elementwise and from the data (u = finfo(dtype).eps / 2, v = 2^-24, tiny =
the type's least subnormal):
  s = x A^T    fp32 sums of K products, then held to 16 bits or more as the next
               product's operand (two parts of the type):
               |ds| <= K v (|x| |A|^T) + 2^-16 |s| + tiny
  y            the shared product may be rounded to the type before the adapters' part
               is added, or take s rounded to the type (half a step, u |s|) into its sum:
               |dy| <= u |y| + u |x W^T| + K v (|x| |W|^T)
                       + c ((|ds| + (u + (r + 4) v) |s|) |B|^T) + tiny
  dx           the same with dy, B for A, A for B, N for K
  dA, dB       sums over the R rows of the adapter:
               |dA| <= u |dA| + c (|dT| + (R + 4) v |T|)^T |x| + tiny
"""
import pytest
import torch

import moe_overlap_b200 as mo

pytestmark = pytest.mark.gpu

V = 2.0 ** -24


def make(M, K, N, L, r, dtype, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).to(dtype).to(device)
    w = (torch.randn(N, K, generator=g) * 0.05).to(dtype).to(device)
    a = (torch.randn(L, r, K, generator=g) / K ** 0.5).to(dtype).to(device)
    b = (torch.randn(L, N, r, generator=g) * 0.1).to(dtype).to(device)
    dy = (torch.randn(M, N, generator=g) * 0.1).to(dtype).to(device)
    scale = (0.5 + torch.rand(L, generator=g)).to(device)
    ids = torch.randint(-1, L, (M,), generator=g).to(device)
    return x, w, a, b, dy, scale, ids


def low(x, A, K, tiny):
    """x A^T in 64 bits and how far the kernels' may be off."""
    s = x @ A.t()
    return s, K * V * (x.abs() @ A.abs().t()) + 2.0 ** -16 * s.abs() + tiny


def reference(x, w, a, b, dy, scale, ids):
    """((value, tolerance) of y, dx, dA, dB) in 64 bits."""
    dt = x.dtype
    u, tiny = torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    x, w, a, b, dy, scale = (t.detach().double() for t in (x, w, a, b, dy, scale))
    (M, K), N, r = x.shape, w.shape[0], a.shape[1]
    y, dx = x @ w.t(), dy @ w
    ty = u * y.abs() + K * V * (x.abs() @ w.abs().t()) + tiny
    tx = u * dx.abs() + N * V * (dy.abs() @ w.abs()) + tiny
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    ta, tb = torch.full_like(a, tiny), torch.full_like(b, tiny)
    for i in range(a.shape[0]):
        rows = (ids == i).nonzero()[:, 0]
        c, R = float(scale[i]), rows.numel()
        s, ds = low(x[rows], a[i], K, tiny)
        t, dt_ = low(dy[rows], b[i].t(), N, tiny)
        y[rows] += c * (s @ b[i].t())
        ty[rows] += c * ((ds + (u + (r + 4) * V) * s.abs()) @ b[i].abs().t())
        dx[rows] += c * (t @ a[i])
        tx[rows] += c * ((dt_ + (u + (r + 4) * V) * t.abs()) @ a[i].abs())
        da[i] = c * (t.t() @ x[rows])
        ta[i] += c * ((dt_ + (R + 4) * V * t.abs()).t() @ x[rows].abs())
        db[i] = c * (dy[rows].t() @ s)
        tb[i] += c * (dy[rows].abs().t() @ (ds + (R + 4) * V * s.abs()))
    return ((y, ty + u * y.abs()), (dx, tx + u * dx.abs()), (da, ta + u * da.abs()),
            (db, tb + u * db.abs()))


def assert_close(got, want):
    value, tol = want
    assert got.shape == value.shape
    bad = ~((got.double() - value).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - value).abs() / tol).max()))


SHAPES = [
    (1, 8, 8, 1, 8, torch.bfloat16), (70, 8, 16, 2, 8, torch.float16), (1, 64, 64, 1, 8, torch.bfloat16), (1, 2048, 256, 4, 16, torch.bfloat16),
    (3, 72, 136, 2, 8, torch.float16), (7, 512, 1000, 5, 24, torch.bfloat16),
    (16, 264, 520, 16, 32, torch.bfloat16), (33, 1000, 72, 3, 64, torch.float16),
    (64, 256, 256, 64, 16, torch.bfloat16), (65, 128, 384, 2, 128, torch.bfloat16),
    (129, 520, 264, 7, 40, torch.float16), (300, 192, 640, 1, 16, torch.bfloat16),
    (777, 320, 200, 40, 56, torch.bfloat16), (2050, 136, 328, 6, 64, torch.float16),
]


@pytest.mark.parametrize("M,K,N,L,r,dtype", SHAPES)
def test_forward_matches_64_bit_reference(cuda_device, M, K, N, L, r, dtype):
    x, w, a, b, dy, scale, ids = make(M, K, N, L, r, dtype, seed=M + r, device=cuda_device)
    y = mo.lora_linear(x, w, a, b, ids, scale=scale)
    mo.check_status(cuda_device, sync=True)
    assert y.dtype == dtype
    assert_close(y, reference(x, w, a, b, dy, scale, ids)[0])
    assert torch.equal(mo.lora_linear(x, w, a, b, ids.to(torch.int32), scale=scale), y)


@pytest.mark.parametrize("M,K,N,L,r,dtype", [
    (900, 256, 520, 9, 16, torch.bfloat16), (515, 136, 264, 30, 128, torch.bfloat16),
    (1290, 520, 136, 6, 72, torch.float16), (256, 64, 512, 1000, 8, torch.bfloat16),
    (300, 192, 256, 5, 64, torch.float16)])
def test_rows_in_runs_and_tiles_of_many_adapters(cuda_device, M, K, N, L, r, dtype):
    """Rows of an adapter together, so that most tiles of 256 rows hold few adapters, with
    one stretch of rows in which every row has another one, and a short last tile."""
    x, w, a, b, dy, scale, _ = make(M, K, N, L, r, dtype, seed=M + L, device=cuda_device)
    ids = torch.arange(M) // 97 % L
    ids[300:420] = torch.arange(len(ids[300:420])) % L
    ids[40:60] = -1
    ids = ids.to(cuda_device)
    for t in (x, a, b):
        t.requires_grad_(True)
    y = mo.lora_linear(x, w, a, b, ids, scale=scale)
    grads = torch.autograd.grad(y, (x, a, b), dy)
    mo.check_status(cuda_device, sync=True)
    for got, want in zip((y, *grads), reference(x, w, a, b, dy, scale, ids)):
        assert_close(got, want)


@pytest.mark.parametrize("M,K,N,L,r,dtype", SHAPES)
def test_gradients_match_64_bit_reference(cuda_device, M, K, N, L, r, dtype):
    x, w, a, b, dy, scale, ids = make(M, K, N, L, r, dtype, seed=M * 3 + r, device=cuda_device)
    for t in (x, a, b):
        t.requires_grad_(True)
    y = mo.lora_linear(x, w, a, b, ids, scale=scale)
    grads = torch.autograd.grad(y, (x, a, b), dy)
    mo.check_status(cuda_device, sync=True)
    for got, want in zip((y, *grads), reference(x, w, a, b, dy, scale, ids)):
        assert_close(got, want)
    y = mo.lora_linear(x, w, a, b, ids, scale=scale)
    for one, two in zip(torch.autograd.grad(y, (x, a, b), dy), grads):
        assert torch.equal(one, two)  # sums in a fixed order


def test_gradients_match_differences(cuda_device):
    """<G, D> against (f(p + hD) - f(p - hD)) / 2h with f = <dy, y> evaluated in 64 bits:
    f is linear in each of x, A and B alone, so the difference is exact up to fp64."""
    M, K, N, L, r = 40, 96, 80, 3, 16
    x, w, a, b, dy, scale, ids = make(M, K, N, L, r, torch.bfloat16, seed=11, device=cuda_device)
    ref = reference(x, w, a, b, dy, scale, ids)
    for t in (x, a, b):
        t.requires_grad_(True)
    grads = torch.autograd.grad(mo.lora_linear(x, w, a, b, ids, scale=scale), (x, a, b), dy)
    g = torch.Generator(device=cuda_device).manual_seed(2)

    def f(x, a, b):
        y = x @ w.double().t()
        for i in range(L):
            m = ids == i
            y[m] += float(scale[i]) * (x[m] @ a[i].t()) @ b[i].t()
        return float((y * dy.double()).sum())

    p = [t.detach().double() for t in (x, a, b)]
    for n in range(3):
        d = torch.randn(p[n].shape, generator=g, device=cuda_device, dtype=torch.float64)
        up, down = list(p), list(p)
        up[n], down[n] = p[n] + d, p[n] - d
        want = (f(*up) - f(*down)) / 2
        tol = float((ref[n + 1][1] * d.abs()).sum()) + 1e-9 * abs(want)
        assert abs(float((grads[n].double() * d).sum()) - want) <= tol


@pytest.mark.parametrize("needs", [(True, False, False), (False, True, False), (False, False, True)])
def test_only_the_gradients_asked_for(cuda_device, needs):
    x, w, a, b, dy, scale, ids = make(20, 64, 72, 2, 8, torch.bfloat16, device=cuda_device)
    ts = (x, a, b)
    for t, n in zip(ts, needs):
        t.requires_grad_(n)
    mo.lora_linear(x, w, a, b, ids, scale=scale).backward(dy)
    ref = reference(x, w, a, b, dy, scale, ids)[1:]
    for t, n, want in zip(ts, needs, ref):
        assert (t.grad is not None) == n
        if n:
            assert_close(t.grad, want)


def test_rows_without_adapter_adapters_without_rows(cuda_device):
    M, K, N, L, r = 50, 128, 136, 4, 16
    x, w, a, b, dy, scale, _ = make(M, K, N, L, r, torch.bfloat16, device=cuda_device)
    none = torch.full((M,), -1, device=cuda_device)
    one = none.clone()
    one[17] = 2
    a[1], b[3] = float("nan"), float("inf")  # adapters without rows: never read into a result
    for ids in (none, one):
        p = [t.clone().requires_grad_(True) for t in (x, a, b)]
        y = mo.lora_linear(p[0], w, p[1], p[2], ids, scale=scale)
        grads = torch.autograd.grad(y, p, dy)
        assert bool(y.isfinite().all())
        for g in grads[1:]:
            for i in range(L):
                if not bool((ids == i).any()):
                    assert bool((g[i] == 0).all())
        keep = [0, 2]
        fix = torch.where(ids == 2, 1, ids)
        for got, want in zip((y, grads[0]), reference(x, w, a[keep], b[keep], dy, scale[keep], fix)):
            assert_close(got, want)


@pytest.mark.parametrize("M,L,dtype", [(40, 4, torch.bfloat16), (700, 4, torch.float16), (700, 12, torch.bfloat16)])
def test_an_adapters_infinities_stay_in_its_rows(cuda_device, M, L, dtype):
    """Requests share tiles of rows, not their adapters: infinities and NaN in two adapters
    change no bit of the other rows, with or without an adapter, nor of the other gradients."""
    x, w, a, b, dy, scale, ids = make(M, 192, 264, L, 16, dtype, seed=L, device=cuda_device)

    def run(a, b, grad):
        p = [t.detach().clone().requires_grad_(grad) for t in (x, a, b)]
        y = mo.lora_linear(p[0], w, p[1], p[2], ids, scale=scale)
        return (y.detach(), *torch.autograd.grad(y, p, dy)) if grad else (y,)

    bad_a, bad_b = a.clone(), b.clone()
    bad_a[1, 3, 5], bad_a[2] = float("inf"), float("nan")
    bad_b[1, 7], bad_b[2, 100, 4] = float("-inf"), float("nan")
    clean_rows = (ids != 1) & (ids != 2)
    others = [i for i in range(L) if i not in (1, 2)]
    for grad in (False, True):
        good, bad = run(a, b, grad), run(bad_a, bad_b, grad)
        assert not bool(bad[0][~clean_rows].isfinite().all())
        for g, h in zip(good[:2], bad[:2]):
            assert torch.equal(g[clean_rows], h[clean_rows])
        for g, h in zip(good[2:], bad[2:]):
            assert torch.equal(g[others], h[others])


def test_backward_passes_may_be_repeated_but_not_differentiated(cuda_device):
    x, w, a, b, dy, scale, ids = make(600, 128, 136, 3, 16, torch.bfloat16, device=cuda_device)
    p = [t.requires_grad_(True) for t in (x, a, b)]
    y = mo.lora_linear(x, w, a, b, ids, scale=scale)
    first = torch.autograd.grad(y, p, dy, retain_graph=True)
    (only_x,) = torch.autograd.grad(y, (x,), 2 * dy, retain_graph=True)
    for one, two in zip(torch.autograd.grad(y, p, dy, retain_graph=True), first):
        assert torch.equal(one, two)
    assert torch.equal(only_x, 2 * first[0])  # powers of two change no rounding
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y, p, dy, create_graph=True)


def test_no_rows(cuda_device):
    x, w, a, b, dy, scale, ids = make(0, 64, 72, 2, 8, torch.bfloat16, device=cuda_device)
    for t in (x, a, b):
        t.requires_grad_(True)
    y = mo.lora_linear(x, w, a, b, ids, scale=scale)
    assert y.shape == (0, 72)
    dx, da, db = torch.autograd.grad(y, (x, a, b), dy)
    assert dx.shape == (0, 64) and bool((da == 0).all()) and bool((db == 0).all())


@pytest.mark.parametrize("M,K,N,r", [(5, 61, 43, 3), (70, 130, 75, 17), (200, 64, 100, 1)])
def test_odd_sizes_are_padded(cuda_device, M, K, N, r):
    x, w, a, b, dy, scale, ids = make(M, K, N, 3, r, torch.bfloat16, seed=r, device=cuda_device)
    for t in (x, a, b):
        t.requires_grad_(True)
    y = mo.lora_linear(x, w, a, b, ids, scale=scale)
    assert y.shape == (M, N)
    grads = torch.autograd.grad(y, (x, a, b), dy)
    for got, want in zip((y, *grads), reference(x, w, a, b, dy, scale, ids)):
        assert_close(got, want)


def test_strided_inputs(cuda_device):
    M, K, N, L, r = 37, 128, 96, 3, 16
    x, w, a, b, dy, scale, ids = make(M, K, N, L, r, torch.bfloat16, device=cuda_device)

    def wide(t, by):  # the same values with wider rows
        big = torch.full((*t.shape[:-1], t.shape[-1] + by), 9.0, dtype=t.dtype, device=t.device)
        big[..., :t.shape[-1]] = t
        return big[..., :t.shape[-1]]

    def run(x, w, a, b, dy):
        p = [t.detach().requires_grad_(True) for t in (x, a, b)]
        y = mo.lora_linear(p[0], w, p[1], p[2], ids, scale=scale)
        return (y, *torch.autograd.grad(y, p, dy))

    ref = run(x, w, a, b, dy)
    for by in (8, 3):
        for one, two in zip(run(wide(x, by), wide(w, by), wide(a, by), wide(b, by), wide(dy, by)), ref):
            assert torch.equal(one, two)
    cols = run(x.t().contiguous().t(), w.t().contiguous().t(), a.transpose(1, 2).contiguous().transpose(1, 2),
               b.transpose(1, 2).contiguous().transpose(1, 2), dy.t().contiguous().t())
    for one, two in zip(cols, ref):
        assert torch.equal(one, two)
    y = mo.lora_linear(x.requires_grad_(True), w, a, b, ids, scale=2.0)
    (dx,) = torch.autograd.grad(y.sum(), (x,))  # an expanded gradient (strides of 0)
    assert_close(dx, reference(x, w, a, b, torch.ones_like(dy), torch.full((L,), 2.0), ids)[1])


def test_bad_ids_count_as_none_and_raise_later(cuda_device):
    x, w, a, b, _, scale, ids = make(40, 64, 72, 3, 8, torch.bfloat16, device=cuda_device)
    bad = ids.clone()
    bad[::7] = 3
    bad[1::7] = -2
    bad[2::7] = 1 << 40
    y = mo.lora_linear(x, w, a, b, bad, scale=scale)
    with pytest.raises(mo.MoeError):
        mo.check_status(cuda_device, sync=True)
    fixed = torch.where((bad < -1) | (bad > 2), -1, bad)
    assert torch.equal(mo.lora_linear(x, w, a, b, fixed, scale=scale), y)


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
@pytest.mark.parametrize("M", [3, 200])
def test_streams_and_graph(cuda_device, M):
    """Calls at once on two streams and a captured training step replayed on new data
    give the bits of a call alone.  A capture while an eager graph of the same leaves
    lives is refused, and leaves the process and the GPU usable."""
    K, N, L, r = 256, 320, 4, 16
    x, w, a, b, dy, scale, ids = make(M, K, N, L, r, torch.bfloat16, seed=1, device=cuda_device)
    x2, ids2 = make(M, K, N, L, r, torch.bfloat16, seed=2, device=cuda_device)[0::6]
    for t in (x, a, b):
        t.requires_grad_(True)

    def step(x, ids):
        y = mo.lora_linear(x, w, a, b, ids, scale=scale)
        return (y.detach(), *torch.autograd.grad(y, (x, a, b), dy))

    want = step(x, ids)
    want2 = step(x2.requires_grad_(True), ids2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            one = step(x, ids)
        with torch.cuda.stream(s2):
            two = step(x2, ids2)
        got.append((one, two))
    torch.cuda.synchronize()
    for one, two in got:
        assert all(torch.equal(p, q) for p, q in zip(one, want))
        assert all(torch.equal(p, q) for p, q in zip(two, want2))
    del got, one, two
    xs, idss = x.detach().clone().requires_grad_(True), ids.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(xs, idss)
    torch.cuda.current_stream().wait_stream(side)
    alive = mo.lora_linear(x, w, a, b, ids, scale=scale)
    with pytest.raises(RuntimeError, match="is alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step(xs, idss)
    assert torch.equal(alive, want[0])
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xs, idss)
    for xi, ii, ref in ((x2, ids2, want2), (x, ids, want)):
        with torch.no_grad():
            xs.copy_(xi)
            idss.copy_(ii)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, ref):
            assert torch.equal(p, q)


@pytest.mark.parametrize("M,N,dtype", [(1, 2048, torch.bfloat16), (5, 6408, torch.float16),
                                       (13, 3208, torch.bfloat16), (29, 8200, torch.bfloat16),
                                       (40, 72, torch.float16), (64, 4000, torch.bfloat16),
                                       (65, 136, torch.bfloat16), (200, 520, torch.float16),
                                       (128, 6400, torch.bfloat16)])
def test_decode_batches_on_streams_and_in_a_graph(cuda_device, M, N, dtype):
    """Few rows without gradients: against 64 bits over the widths of the weight, two
    calls at once, a replayed capture, and in inference mode."""
    K, L, r = 328, 3, 24
    x, w, a, b, dy, scale, ids = make(M, K, N, L, r, dtype, seed=M, device=cuda_device)
    x2, ids2 = make(M, K, N, L, r, dtype, seed=M + 1, device=cuda_device)[0::6]
    ref, ref2 = (mo.lora_linear(p, w, a, b, i, scale=scale) for p, i in ((x, ids), (x2, ids2)))
    assert_close(ref, reference(x, w, a, b, dy, scale, ids)[0])
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            one = mo.lora_linear(x, w, a, b, ids, scale=scale)
        with torch.cuda.stream(s2), torch.inference_mode():
            two = mo.lora_linear(x2, w, a, b, ids2, scale=scale)
        got.append((one, two))
    torch.cuda.synchronize()
    assert all(torch.equal(one, ref) and torch.equal(two, ref2) for one, two in got)
    xs, idss = x.clone(), ids.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mo.lora_linear(xs, w, a, b, idss, scale=scale)
    for p, i, want in ((x2, ids2, ref2), (x, ids, ref)):
        xs.copy_(p)
        idss.copy_(i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_a_decode_step_with_adapters_then_the_experts(cuda_device):
    """As they are used together: the projection before the experts with each request's
    adapter, then the routed experts, for a decode batch with padding."""
    T, H, F, E, L = 9, 256, 384, 8, 4
    x, w, a, b, _, scale, ids = make(T, H, H, L, 16, torch.bfloat16, seed=5, device=cuda_device)
    g = torch.Generator().manual_seed(3)
    rw = (torch.randn(E, H, generator=g) * 0.05).to(torch.bfloat16).to(cuda_device)
    w1 = (torch.randn(E, F, H, generator=g) * 0.05).to(torch.bfloat16).to(cuda_device)
    w2 = (torch.randn(E, H, F, generator=g) * 0.05).to(torch.bfloat16).to(cuda_device)
    ids[-1] = -1
    y = mo.lora_linear(x, w, a, b, ids, scale=scale)
    assert_close(y, reference(x, w, a, b, torch.zeros(T, H, device=cuda_device), scale, ids)[0])
    out, idx, wt = mo.moe_few_tokens(y, rw, w1, w2, 2, renormalize=True)
    idx[-1] = -1
    padded = mo.experts_few_tokens(y, w1, w2, idx, wt)
    assert torch.equal(padded[:-1], out[:-1]) and bool((padded[-1] == 0).all())
    from tests.test_few_tokens_gpu import experts64

    want, tol = experts64(y, w1, w2, idx, wt.double())
    assert bool(((padded.double() - want).abs() <= tol).all())


def test_rows_past_32_bit_offsets(cuda_device):
    """The last rows of x start past 2^31 elements."""
    M, K, N, L, r = 262152 + 300, 8192, 8, 2, 8
    _, w, a, b, _, scale, _ = make(1, K, N, L, r, torch.bfloat16, seed=3, device=cuda_device)
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=cuda_device)
    at = [0, 5, M // 2, M - 300, M - 1]
    x[at] = make(len(at), K, N, L, r, torch.bfloat16, seed=4, device=cuda_device)[0]
    ids = torch.full((M,), -1, device=cuda_device)
    ids[at] = torch.tensor([0, 1, -1, 1, 0], device=cuda_device)
    dy = torch.zeros(M, N, dtype=torch.bfloat16, device=cuda_device)
    dy[at] = make(len(at), K, N, L, r, torch.bfloat16, seed=4, device=cuda_device)[4]
    for t in (x, a, b):
        t.requires_grad_(True)
    y = mo.lora_linear(x, w, a, b, ids, scale=scale)
    dx, da, db = torch.autograd.grad(y, (x, a, b), dy)
    mo.check_status(cuda_device, sync=True)
    want = reference(x[at], w, a, b, dy[at], scale, ids[at])
    for got, ref in zip((y[at], dx[at], da, db), want):
        assert_close(got, ref)
    rest = torch.ones(M, dtype=torch.bool, device=cuda_device)
    rest[at] = False
    assert not bool(y[rest].any()) and not bool((dx[M - 299:M - 1] != 0).any())


def test_refusals(cuda_device):
    x, w, a, b, _, scale, ids = make(6, 64, 72, 3, 8, torch.bfloat16, device=cuda_device)
    f = mo.lora_linear
    for call, match in (
            (lambda: f(x.float(), w, a, b, ids), "bf16/fp16"), (lambda: f(x, w.half(), a, b, ids), "weight must be"),
            (lambda: f(x, w, a.cpu(), b, ids), "lora_a must be"), (lambda: f(x, w, a, b.float(), ids), "lora_b must be"),
            (lambda: f(x[0], w, a, b, ids), "Shapes"), (lambda: f(x, w, a, b[:2], ids), "Shapes"),
            (lambda: f(x, w, a[:, :, :56], b, ids), "Shapes"), (lambda: f(x, w.t(), a, b, ids), "Shapes"),
            (lambda: f(x, w, a, b, ids[:5]), "adapter_ids"), (lambda: f(x, w, a, b, ids.float()), "adapter_ids"),
            (lambda: f(x, w, a, b, ids.cpu()), "adapter_ids"),
            (lambda: f(x, w, a, b, ids, scale=scale[:2]), "scale"), (lambda: f(x, w, a, b, ids, scale=ids[:3]), "scale"),
            (lambda: f(x, w, a.new_zeros(3, 136, 64), b.new_zeros(3, 72, 136), ids), "ranks"),
            (lambda: f(x, w, a[:0], b[:0], ids), "adapters"),
            (lambda: f(x, w.clone().requires_grad_(True), a, b, ids), "frozen"),
            (lambda: f(x, w, a, b, ids, scale=scale.clone().requires_grad_(True)), "no gradient")):
        with pytest.raises(ValueError, match=match):
            call()
    with torch.no_grad():  # nothing asks for those gradients here
        assert f(x, w.clone().requires_grad_(True), a, b, ids).shape == (6, 72)
    mo.check_status(cuda_device, sync=True)


@pytest.mark.parametrize("M,K,N,L,r,dtype", [
    (66, 1032, 264, 3, 8, torch.bfloat16), (200, 264, 1048, 8, 40, torch.float16),
    (300, 1040, 1104, 1, 128, torch.bfloat16), (700, 2056, 1000, 8, 64, torch.float16),
    (515, 1096, 1160, 20, 16, torch.bfloat16), (1500, 1024, 1100, 9, 24, torch.bfloat16)])
@pytest.mark.parametrize("runs", [False, True])
def test_few_tiles_of_long_contractions(cuda_device, M, K, N, L, r, dtype, runs):
    """Few tiles of the output: their contraction over K (backward: over N) is split, and
    the adapters of a tile with it; rows of an adapter together or in any order."""
    x, w, a, b, dy, scale, ids = make(M, K, N, L, r, dtype, seed=M + K, device=cuda_device)
    if runs:
        ids = torch.sort(ids).values
    for t in (x, a, b):
        t.requires_grad_(True)
    y = mo.lora_linear(x, w, a, b, ids, scale=scale)
    grads = torch.autograd.grad(y, (x, a, b), dy)
    mo.check_status(cuda_device, sync=True)
    for got, want in zip((y, *grads), reference(x, w, a, b, dy, scale, ids)):
        assert_close(got, want)
    y2 = mo.lora_linear(x, w, a, b, ids, scale=scale)
    for one, two in zip((y2, *torch.autograd.grad(y2, (x, a, b), dy)), (y, *grads)):
        assert torch.equal(one, two)  # sums in a fixed order


@pytest.mark.parametrize("M,K,N,L,r,dtype", [
    (600, 264, 520, 14, 32, torch.bfloat16), (600, 136, 264, 16, 8, torch.float16),
    (513, 200, 72, 12, 16, torch.bfloat16), (700, 320, 264, 8, 24, torch.float16),
    (300, 1040, 1032, 16, 32, torch.bfloat16), (260, 72, 1000, 17, 32, torch.float16),
    (400, 72, 264, 8, 72, torch.bfloat16), (400, 72, 264, 9, 40, torch.bfloat16)])
def test_stages_shared_by_adapters(cuda_device, M, K, N, L, r, dtype):
    """Every adapter in every tile of rows: as many as the shared product takes, and one more."""
    x, w, a, b, dy, scale, _ = make(M, K, N, L, r, dtype, seed=L * r, device=cuda_device)
    ids = (torch.arange(M) % (L + 1) - 1).to(cuda_device)
    for t in (x, a, b):
        t.requires_grad_(True)
    y = mo.lora_linear(x, w, a, b, ids, scale=scale)
    grads = torch.autograd.grad(y, (x, a, b), dy)
    mo.check_status(cuda_device, sync=True)
    for got, want in zip((y, *grads), reference(x, w, a, b, dy, scale, ids)):
        assert_close(got, want)


@pytest.mark.parametrize("M,K,N", [(300, 1040, 264), (300, 264, 1040), (900, 1032, 1032)])
def test_infinities_with_split_contractions(cuda_device, M, K, N):
    x, w, a, b, dy, scale, ids = make(M, K, N, 5, 16, torch.bfloat16, seed=M, device=cuda_device)

    def run(a, b):
        p = [t.detach().clone().requires_grad_() for t in (x, a, b)]
        y = mo.lora_linear(p[0], w, p[1], p[2], ids, scale=scale)
        return (y.detach(), *torch.autograd.grad(y, p, dy))

    bad_a, bad_b = a.clone(), b.clone()
    bad_a[1, 3, 5], bad_b[2, 7] = float("inf"), float("nan")
    clean_rows = (ids != 1) & (ids != 2)
    good, bad = run(a, b), run(bad_a, bad_b)
    assert not bool(bad[0][~clean_rows].isfinite().all())
    for g, h in zip(good[:2], bad[:2]):
        assert torch.equal(g[clean_rows], h[clean_rows])
    for g, h in zip(good[2:], bad[2:]):
        assert torch.equal(g[[0, 3, 4]], h[[0, 3, 4]])


@pytest.mark.parametrize("M", [1, 40, 300])
def test_broadcast_inputs_and_shared_adapters(cuda_device, M):
    """An output summed (a gradient of stride 0), one adapter expanded over all requests, and
    adapters that stand twice in one graph."""
    x, w, a, b, _, scale, ids = make(M, 264, 264, 4, 16, torch.bfloat16, seed=M, device=cuda_device)
    one = a[:1].clone().requires_grad_()
    x.requires_grad_()
    y = mo.lora_linear(x, w, one.expand_as(a), b, ids, scale=scale)
    dx, da = torch.autograd.grad(y.sum(), (x, one))
    want = reference(x, w, one.expand_as(a), b, torch.ones_like(y), scale, ids)
    assert_close(dx, want[1])
    per_adapter, tol = want[2]
    # each adapter's gradient is rounded, then their sum (three additions and a rounding of it)
    u = torch.finfo(a.dtype).eps / 2
    assert_close(da[0], (per_adapter.sum(0), tol.sum(0) + 4 * u * per_adapter.abs().sum(0)))

    a.requires_grad_(), b.requires_grad_()
    h = mo.lora_linear(x.detach(), w, a, b, ids, scale=scale)
    y = mo.lora_linear(h, w, a, b, ids, scale=scale)
    both = torch.autograd.grad(y, (a, b), torch.ones_like(y))
    h2 = h.detach().requires_grad_()
    second = torch.autograd.grad(mo.lora_linear(h2, w, a, b, ids, scale=scale), (h2, a, b), torch.ones_like(y))
    first = torch.autograd.grad(mo.lora_linear(x.detach(), w, a, b, ids, scale=scale), (a, b), second[0])
    for got, p, q in zip(both, first, second[1:]):
        assert torch.equal(got, p + q)
