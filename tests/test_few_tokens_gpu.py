"""GPU parity of the few-token experts layer against a plain evaluation in 64 bits.

Tolerances, elementwise and from the data (u = finfo(dtype).eps / 2, v = 2^-24):
  a = x W1^T       fp32 sums of H products:          |da| <= H v (|x| |W1|^T)
  h = gelu(a)      |gelu'| < 1.13, rounded to dtype: |dh| <= 1.13 |da| + (u + 8 v) |h|
                   (8 v: erff and the two products around it) + the type's least
                   subnormal
  y = h W2^T       |dy| <= |dh| |W2|^T + F v (|h| |W2|^T)
  out = sum w y    |dout| <= sum w (|dy| + (k + 4) v |y|) + sum |dw| |y| + u |out|
                   (+ the least subnormal)
  w                expf (2 ulp), a sum of E of them and two divisions: |dw| <= (E + 16) 2 v w
The experts chosen have to be the reference's: the gate's logits are held in 64 bits.
"""
import pytest
import torch

import moe_overlap_b200 as mo

pytestmark = pytest.mark.gpu

V = 2.0 ** -24


def make(T, E, H, F, dtype, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g).to(dtype).to(device)
    rw = (torch.randn(E, H, generator=g) * 0.05).to(dtype).to(device)
    w1 = (torch.randn(E, F, H, generator=g) * 0.05).to(dtype).to(device)
    w2 = (torch.randn(E, H, F, generator=g) * 0.05).to(dtype).to(device)
    return x, rw, w1, w2


def route64(x, rw, bias, k, renorm):
    z = x.double() @ rw.double().t()
    if bias is not None:
        z = z + bias.double()
    p = torch.softmax(z, dim=1)
    idx = z.sort(dim=1, descending=True, stable=True).indices[:, :k]
    w = p.gather(1, idx)
    return idx, w / w.sum(dim=1, keepdim=True) if renorm else w


def experts64(x, w1, w2, idx, w, dw_rel=0.0):
    """(out, tolerance) in 64 bits; slots of -1 add nothing."""
    T, H = x.shape
    E, F, _ = w1.shape
    u, tiny = torch.finfo(x.dtype).eps / 2, torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    out = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    tol = torch.zeros_like(out)
    k = idx.shape[1]
    for t in range(T):
        for j in range(k):
            e = int(idx[t, j])
            if e < 0:
                continue
            xd, a1, a2 = x[t].double(), w1[e].double(), w2[e].double()
            a = a1 @ xd
            h = torch.nn.functional.gelu(a)
            da = H * V * (a1.abs() @ xd.abs())
            dh = 1.13 * da + (u + 8 * V) * h.abs() + tiny
            y = a2 @ h
            dy = a2.abs() @ dh + F * V * (a2.abs() @ h.abs())
            wt = float(w[t, j])
            out[t] += wt * y
            tol[t] += abs(wt) * (dy + (k + 4) * V * y.abs()) + dw_rel * abs(wt) * y.abs()
    return out, tol + u * out.abs() + tiny


def assert_close(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


@pytest.mark.parametrize("T,E,H,F,k,renorm,bias,dtype", [
    (1, 16, 256, 512, 2, False, False, torch.bfloat16),
    (1, 1, 8, 8, 1, True, False, torch.bfloat16),
    (2, 3, 24, 40, 3, False, True, torch.float16),
    (5, 8, 512, 1024, 2, True, False, torch.float16),
    (7, 4, 1000, 136, 1, False, True, torch.bfloat16),
    (9, 17, 136, 1000, 4, True, True, torch.bfloat16),
    (17, 5, 264, 72, 5, False, False, torch.bfloat16),
    (31, 256, 64, 16, 8, True, False, torch.float16),
    (64, 16, 512, 256, 2, True, False, torch.bfloat16),
    (65, 2, 128, 264, 2, True, False, torch.bfloat16),
    (128, 40, 72, 128, 16, False, True, torch.bfloat16),
    (128, 3, 648, 328, 1, False, False, torch.float16),
])
def test_moe_few_tokens_matches_64_bit_reference(cuda_device, T, E, H, F, k, renorm, bias, dtype):
    x, rw, w1, w2 = make(T, E, H, F, dtype, seed=T + E + k, device=cuda_device)
    b = -0.3 * torch.arange(E, dtype=torch.float32, device=cuda_device) if bias else None
    out, idx, w = mo.moe_few_tokens(x, rw, w1, w2, k, router_bias=b, renormalize=renorm)
    mo.check_status(cuda_device, sync=True)
    want_i, want_w = route64(x, rw, b, k, renorm)
    assert torch.equal(idx, want_i)
    rel = (E + 16) * 2 * V
    assert bool(((w.double() - want_w).abs() <= rel * want_w + 1e-38).all())
    want, tol = experts64(x, w1, w2, want_i, want_w, dw_rel=rel)
    assert out.dtype == dtype and out.shape == (T, H)
    assert_close(out, want, tol)


@pytest.mark.parametrize("T,k,dtype", [(1, 1, torch.bfloat16), (33, 2, torch.float16), (128, 4, torch.bfloat16)])
def test_given_routing_with_padding_repeats_and_one_hot_expert(cuda_device, T, k, dtype):
    """Rows of -1, half-routed rows, the same expert twice in a row, and one expert
    that takes most slots (several blocks of rows of one expert)."""
    E, H, F = 6, 136, 200
    x, _, w1, w2 = make(T, E, H, F, dtype, seed=3, device=cuda_device)
    g = torch.Generator().manual_seed(1)
    idx = torch.randint(0, E, (T, k), generator=g)
    idx[torch.rand(T, k, generator=g) < 0.6] = 4  # the hot expert, repeated within rows too
    idx[torch.rand(T, k, generator=g) < 0.2] = -1
    idx[T // 2] = -1
    w = torch.rand(T, k, generator=g)
    w[0, 0] = 0.0
    idx, w = idx.to(cuda_device), w.to(cuda_device)
    x[T // 2] = float("nan")  # a padding row's values must not matter
    out = torch.full((T, H + 8), 7.0, dtype=dtype, device=cuda_device)
    got = mo.experts_few_tokens(x, w1, w2, idx, w, out=out[:, :H])
    mo.check_status(cuda_device, sync=True)
    assert got.data_ptr() == out.data_ptr()
    want, tol = experts64(x, w1, w2, idx, w)
    assert_close(got, want, tol)
    assert bool((got[T // 2] == 0).all())
    assert bool((out[:, H:] == 7.0).all())  # columns behind the view stay as they were
    again = mo.experts_few_tokens(x, w1, w2, idx.to(torch.int32), w)
    assert torch.equal(again, got)


def test_all_slots_unrouted_gives_zeros(cuda_device):
    x, _, w1, w2 = make(5, 3, 64, 64, torch.bfloat16, device=cuda_device)
    out = torch.full_like(x, 3.0)
    mo.experts_few_tokens(x, w1, w2, torch.full((5, 2), -1, device=cuda_device),
                          torch.ones(5, 2, device=cuda_device), out=out)
    assert bool((out == 0).all())


def test_no_tokens(cuda_device):
    x, rw, w1, w2 = make(0, 3, 64, 64, torch.bfloat16, device=cuda_device)
    out, idx, w = mo.moe_few_tokens(x, rw, w1, w2, 2)
    assert out.shape == (0, 64) and idx.shape == (0, 2) and w.shape == (0, 2)


def test_unused_experts_weights_and_rows_do_not_reach_the_output(cuda_device):
    """NaN and inf in the weights of experts that no token takes change nothing."""
    x, _, w1, w2 = make(4, 4, 64, 72, torch.bfloat16, device=cuda_device)
    idx = torch.tensor([[0, 2], [2, 0], [2, 2], [0, -1]], device=cuda_device)
    w = torch.rand(4, 2, device=cuda_device)
    clean = mo.experts_few_tokens(x, w1, w2, idx, w)
    w1[1], w2[1], w1[3], w2[3] = float("nan"), float("inf"), float("-inf"), float("nan")
    assert torch.equal(mo.experts_few_tokens(x, w1, w2, idx, w), clean)


def test_ties_and_nonfinite_logits(cuda_device):
    x, rw, w1, w2 = make(3, 6, 64, 32, torch.bfloat16, seed=8, device=cuda_device)
    rw[4] = rw[1]
    rw[5] = rw[1]
    x[0] = 8.0 * rw[1] / rw[1].norm()
    _, idx, w = mo.moe_few_tokens(x, rw, w1, w2, 2)
    assert idx[0].tolist() == [1, 4]
    assert float(w[0, 0]) == float(w[0, 1])
    x[2, 0] = float("nan")
    out, idx, w = mo.moe_few_tokens(x, rw, w1, w2, 2)
    assert idx[2].tolist() == [0, 1] and bool(w[2].isnan().all()) and bool(out[2].isnan().all())
    assert bool(out[:2].isfinite().all())
    bias = torch.tensor([0.0, -float("inf"), 0.0, -float("inf"), 0.0, 0.0], device=cuda_device)
    _, idx, w = mo.moe_few_tokens(x[:2], rw, w1, w2, 5, router_bias=bias)
    assert set(idx[0, :4].tolist()) == {0, 2, 4, 5} and int(idx[0, 4]) == 1 and float(w[0, 4]) == 0.0


def test_strided_views_and_weight_strides(cuda_device):
    """Row strides wider than the rows, experts further apart than their rows."""
    T, E, H, F = 6, 4, 128, 96
    x, rw, w1, w2 = make(T, E, H, F, torch.bfloat16, seed=2, device=cuda_device)
    ref = mo.moe_few_tokens(x, rw, w1, w2, 2)
    xs = torch.zeros(T, H + 24, dtype=x.dtype, device=cuda_device)
    xs[:, 16:16 + H] = x
    big1 = torch.zeros(E, F + 3, H + 8, dtype=x.dtype, device=cuda_device)
    big2 = torch.zeros(E, H + 1, F + 16, dtype=x.dtype, device=cuda_device)
    big1[:, :F, :H], big2[:, :H, :F] = w1, w2
    got = mo.moe_few_tokens(xs[:, 16:16 + H], rw, big1[:, :F, :H], big2[:, :H, :F], 2)
    for a, b in zip(got, ref):
        assert torch.equal(a, b)
    odd = torch.zeros(T, H + 1, dtype=x.dtype, device=cuda_device)  # rows off 16 bytes: copied
    odd[:, 1:] = x
    assert torch.equal(mo.moe_few_tokens(odd[:, 1:], rw, w1, w2, 2)[0], ref[0])


def test_bad_expert_ids_count_as_unrouted_and_raise_later(cuda_device):
    x, _, w1, w2 = make(3, 4, 64, 64, torch.bfloat16, device=cuda_device)
    w = torch.ones(3, 2, device=cuda_device)
    idx = torch.tensor([[0, 4], [1, -7], [2, 1 << 40]], device=cuda_device)
    got = mo.experts_few_tokens(x, w1, w2, idx, w)
    with pytest.raises(mo.MoeError):
        mo.check_status(cuda_device, sync=True)
    idx[:, 1] = -1
    assert torch.equal(mo.experts_few_tokens(x, w1, w2, idx, w), got)


def test_streams_graph_and_repeatability(cuda_device):
    """Two calls at once on two streams, and a captured call replayed on new inputs,
    give the bits of a call alone."""
    T, E, H, F = 13, 8, 512, 768
    x, rw, w1, w2 = make(T, E, H, F, torch.bfloat16, seed=4, device=cuda_device)
    x2 = make(T, E, H, F, torch.bfloat16, seed=5, device=cuda_device)[0]
    ref, ref2 = mo.moe_few_tokens(x, rw, w1, w2, 2), mo.moe_few_tokens(x2, rw, w1, w2, 2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            a = mo.moe_few_tokens(x, rw, w1, w2, 2)
        with torch.cuda.stream(s2):
            b = mo.moe_few_tokens(x2, rw, w1, w2, 2)
        got.append((a, b))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a[0], ref[0]) and torch.equal(b[0], ref2[0]) and torch.equal(a[1], ref[1])
    xs = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, idx, w = mo.moe_few_tokens(xs, rw, w1, w2, 2)
    for src, want in ((x2, ref2), (x, ref), (x2, ref2)):
        xs.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(idx, want[1]) and torch.equal(w, want[2])


def test_layer_forward_few_agrees_with_the_layer(cuda_device):
    """The layer's own path on the same routing: both round h and the output once to
    bf16 and sum in fp32, so they differ by what two such evaluations may."""
    from moe_overlap_b200.layer import MoELayer

    T, E, H, F = 24, 8, 256, 512
    layer = MoELayer(H, F, E, 2, renormalize=True, micro_batch_size=64).init_random(std=0.05, seed=1)
    try:
        x = make(T, E, H, F, torch.bfloat16, seed=6, device=cuda_device)[0]
        routing = layer.route(x)
        want, _ = layer(x, routing=routing)
        got, idx, w = layer.forward_few(x, routing=(routing[1], routing[2]))
        ref, tol = experts64(x, layer.w1, layer.w2, routing[1], routing[2])
        assert_close(got, ref, tol)
        # the exchange path also rounds each expert's row to bf16 before its weighted sum
        u = torch.finfo(torch.bfloat16).eps / 2
        rows = torch.zeros_like(ref)
        for t in range(T):
            for j in range(2):
                e = int(routing[1][t, j])
                h = torch.nn.functional.gelu(layer.w1[e].double() @ x[t].double())
                rows[t] += float(routing[2][t, j]) * (layer.w2[e].double() @ h).abs()
        assert_close(got, want.double(), 2 * tol + u * rows)
        out, idx, w = layer.forward_few(x)
        want_i, want_w = route64(x, layer.router_w, None, 2, True)
        assert torch.equal(idx, want_i)
        ref, tol = experts64(x, layer.w1, layer.w2, want_i, want_w, dw_rel=(E + 16) * 2 * V)
        assert_close(out, ref, tol)
    finally:
        layer.close()


def test_weights_past_32_bit_offsets(cuda_device):
    """The last expert's weights start past 2^31 elements."""
    E, H, F = 256, 4096, 2064
    w1 = torch.zeros(E, F, H, dtype=torch.bfloat16, device=cuda_device)
    w2 = torch.zeros(E, H, F, dtype=torch.bfloat16, device=cuda_device)
    assert w1[E - 1].storage_offset() > 2 ** 31
    x, _, a, b = make(2, 2, H, F, torch.bfloat16, seed=9, device=cuda_device)
    w1[E - 1], w2[E - 1], w1[0], w2[0] = a[0], b[0], a[1], b[1]
    idx = torch.tensor([[E - 1, 0], [0, E - 1]], device=cuda_device)
    w = torch.rand(2, 2, device=cuda_device)
    got = mo.experts_few_tokens(x, w1, w2, idx, w)
    want, tol = experts64(x, a, b, torch.where(idx == 0, 1, 0), w)
    assert_close(got, want, tol)


def test_refusals(cuda_device):
    x, rw, w1, w2 = make(4, 4, 64, 72, torch.bfloat16, device=cuda_device)
    idx = torch.zeros(4, 2, dtype=torch.int64, device=cuda_device)
    w = torch.zeros(4, 2, device=cuda_device)
    few, given = mo.moe_few_tokens, mo.experts_few_tokens
    for call, match in (
            (lambda: few(x.float(), rw, w1, w2, 2), "bf16/fp16"),
            (lambda: few(x, rw.half(), w1, w2, 2), "router_w must be"),
            (lambda: few(x, rw, w1.half(), w2, 2), "w1 must be"),
            (lambda: few(x, rw, w1, w2.cpu(), 2), "w2 must be"),
            (lambda: few(x, rw, w1, w2.transpose(1, 2).contiguous(), 2), "Shapes"),
            (lambda: few(x, rw, w1, w2, 0), "top_k"), (lambda: few(x, rw, w1, w2, 5), "top_k"),
            (lambda: few(x, rw, w1, w2, 2, router_bias=torch.zeros(3, device=cuda_device)), "bias"),
            (lambda: few(x, rw, w1, w2, 2, out=torch.empty(3, 64, dtype=x.dtype, device=cuda_device)), "out"),
            (lambda: few(x, rw, w1, w2, 2, out=torch.empty(4, 64, device=cuda_device)), "out"),
            (lambda: few(x, rw, w1, w2, 2, out=torch.empty(64, 4, dtype=x.dtype, device=cuda_device).t()), "out"),
            (lambda: few(x, rw, w1[:, :, ::2], w2[:, ::2], 2), "Shapes"),
            (lambda: given(x, w1.transpose(1, 2).contiguous().transpose(1, 2), w2, idx, w), "unit-stride"),
            (lambda: given(x[:, :60], w1[:, :, :60], w2[:, :60], idx, w), "multiples of 8"),
            (lambda: given(x, w1[:1].expand(4, 72, 64), w2, idx, w), "one matrix behind another"),
            (lambda: given(x.repeat(33, 1), w1, w2, idx.repeat(33, 1), w.repeat(33, 1)), "at most 128"),
            (lambda: given(x, w1, w2, idx.cpu(), w), "must be on"),
            (lambda: given(x, w1, w2, idx.float(), w), "int64 or int32")):
        with pytest.raises(ValueError, match=match):
            call()
    mo.check_status(cuda_device, sync=True)
    from moe_overlap_b200.layer import MoELayer

    layer = MoELayer(64, 72, 4, 2, micro_batch_size=16, expert_placement=[1, 0, 3, 2])
    try:
        with pytest.raises(ValueError, match="contiguous placement"):
            layer.forward_few(x)
    finally:
        layer.close()


@pytest.mark.parametrize("T,E,H,F,k,dtype", [
    (100, 3, 264, 520, 3, torch.bfloat16), (128, 5, 136, 328, 4, torch.float16),
    (17, 2, 1032, 72, 2, torch.bfloat16), (8, 4, 264, 136, 2, torch.float16),
    (8, 4, 264, 136, 3, torch.bfloat16), (9, 40, 520, 264, 2, torch.bfloat16),
    (100, 3, 1032, 3208, 3, torch.bfloat16), (128, 40, 1024, 264, 5, torch.float16),
    (49, 9, 1080, 1096, 8, torch.bfloat16)])
def test_many_slots_an_expert(cuda_device, T, E, H, F, k, dtype):
    """Several groups of slots an expert, the last one short, and both row blocks' limits."""
    test_moe_few_tokens_matches_64_bit_reference(cuda_device, T, E, H, F, k, True, True, dtype)
