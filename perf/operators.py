"""Cases of the two serving and fine-tuning operators that stand beside the layer's
own products, with their plain torch forms.

``few``   A whole routed-experts layer for a few tokens: gate product, softmax, top-k,
          up-projection with exact GELU, down-projection, weighted sum
          (``moe_few_tokens``), or the same from a routing that the caller has
          (``experts_few_tokens``; -1 in a slot routes it nowhere, as in the exchange).
``lora``  A projection that all requests share with the low-rank adapter of each row's
          request beside it (``lora_linear``): forward, and forward with backward.

The plain forms hold every sum in 32 bits (the gate's logits in 64: a choice of
experts hangs on them), and round once at the end.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One user's next token on the repository's 16-expert layer (hidden 2048, ffn 4096):
        # two experts' weights are all there is to read, latency is what counts.
        dict(name="few_t1_e16", kind="few", T=1, E=16, H=2048, F=4096, k=2, dtype="bf16",
             renorm=False, bias=False, given=False),
        # The smallest layer (8 experts, 512 x 1024, half precision), an odd handful of tokens.
        dict(name="few_t5_small_fp16", kind="few", T=5, E=8, H=512, F=1024, k=2, dtype="fp16",
             renorm=True, bias=False, given=False),
        # A decode batch on the layer with the biased gate (hidden 2048, ffn 8192).
        dict(name="few_t16_bias", kind="few", T=16, E=16, H=2048, F=8192, k=2, dtype="bf16",
             renorm=True, bias=True, given=False),
        # Many small experts, eight a token, an odd batch.
        dict(name="few_t37_e64_k8", kind="few", T=37, E=64, H=2048, F=1024, k=8, dtype="bf16",
             renorm=True, bias=False, given=False),
        # The largest decode batch, padded: the caller routes, and a quarter of the rows are
        # padding (every slot -1).
        dict(name="few_t64_given_padded", kind="few", T=64, E=16, H=2048, F=8192, k=2,
             dtype="bf16", renorm=False, bias=False, given=True),
        # One token through a square projection with adapters: the smallest call.
        dict(name="lora_m1", kind="lora", M=1, K=2048, N=2048, L=8, r=16, dtype="bf16",
             order="mixed", train=False),
        # A decode batch, every row its own request's adapter, some without one.
        dict(name="lora_m48_decode", kind="lora", M=48, K=2048, N=8192, L=32, r=16, dtype="bf16",
             order="mixed", train=False),
        # A short ragged prompt batch in half precision, rows of the requests interleaved.
        dict(name="lora_m1003_fp16", kind="lora", M=1003, K=2048, N=1000, L=5, r=64, dtype="fp16",
             order="mixed", train=False),
        # A prompt batch: each request's rows together (batch 8 x 1024 tokens).
        dict(name="lora_m8192_prompt", kind="lora", M=8192, K=2048, N=8192, L=16, r=32,
             dtype="bf16", order="runs", train=False),
        # Fine-tuning several adapters on a small ragged batch, half precision.
        dict(name="lora_m515_train_fp16", kind="lora", M=515, K=512, N=1024, L=3, r=8, dtype="fp16",
             order="mixed", train=True),
        # Fine-tuning, one step of batch 2 x 2048 tokens on a square projection.
        dict(name="lora_m4096_train", kind="lora", M=4096, K=2048, N=2048, L=4, r=16, dtype="bf16",
             order="runs", train=True),
        # The largest step: batch 8 x 2048 tokens through the up-projection.
        dict(name="lora_m16384_train", kind="lora", M=16384, K=2048, N=8192, L=8, r=64,
             dtype="bf16", order="runs", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Sizes over their logarithm; feature sizes are multiples of 8 (what a 16-byte row
    start needs), token counts and expert counts are anything."""
    if rng.random() < 0.45:
        E = _log(rng, 4, 64)
        k = rng.randint(1, min(8, E))
        H = 8 * _log(rng, 32, 512)
        F = 8 * _log(rng, 64, 1024)
        # no more weights than the largest listed layer (16 experts, 2048 x 8192)
        F = max(64, min(F, 8 * ((16 * 2048 * 8192) // (E * H * 8))))
        return dict(kind="few", T=_log(rng, 1, 64), E=E, H=H, F=F, k=k,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), renorm=rng.random() < 0.5,
                    bias=rng.random() < 0.3, given=rng.random() < 0.3)
    train = rng.random() < 0.4
    return dict(kind="lora", M=_log(rng, 16 if train else 1, 16384 if train else 8192),
                K=8 * _log(rng, 32, 256), N=8 * _log(rng, 32, 1024), L=_log(rng, 1, 32),
                r=8 * _log(rng, 1, 8), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                order=rng.choice(["mixed", "runs"]), train=train)


# ---------------------------------------------------------------------- inputs --
def _rows_to_adapters(g, M, L, order):
    """An adapter id for each row, -1 (no adapter) for about an eighth of them; "runs"
    keeps the rows of a request together, in runs of uneven length."""
    dev = g.device
    if order == "runs":
        cuts = torch.rand(max(2 * L, 2), generator=g, device=dev).sort().values
        at = torch.searchsorted(cuts, (torch.arange(M, device=dev) + 0.5) / M)
        ids = torch.randint(0, L, (cuts.numel() + 1,), generator=g, device=dev)
        keep = torch.rand(cuts.numel() + 1, generator=g, device=dev) >= 0.125
        return torch.where(keep, ids, -1)[at]
    ids = torch.randint(0, L, (M,), generator=g, device=dev)
    return torch.where(torch.rand(M, generator=g, device=dev) >= 0.125, ids, -1)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = _DT[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).mul_(std).to(dt)

    s = dict(case)
    if case["kind"] == "few":
        T, E, H, F, k = (case[n] for n in ("T", "E", "H", "F", "k"))
        s["x"] = normal(T, H)
        s["router_w"] = normal(E, H, std=0.02)
        s["router_b"] = None
        if case["bias"]:  # a gate whose experts are unevenly popular
            s["router_b"] = -0.5 * torch.arange(1, E + 1, device=dev, dtype=torch.float32).log()
        s["w1"] = normal(E, F, H, std=0.02)
        s["w2"] = normal(E, H, F, std=0.02)
        if case["given"]:
            idx = torch.rand(T, E, generator=g, device=dev).argsort(dim=1)[:, :k].contiguous()
            w = torch.rand(T, k, generator=g, device=dev)
            pad = torch.arange(T, device=dev) >= T - T // 4
            s["idx"] = torch.where(pad[:, None], -1, idx)
            s["w"] = w / w.sum(dim=1, keepdim=True)
        return s
    M, K, N, L, r = (case[n] for n in ("M", "K", "N", "L", "r"))
    s["x"] = normal(M, K)
    s["weight"] = normal(N, K, std=0.02)
    s["a"] = normal(L, r, K, std=1.0 / math.sqrt(K))
    s["b"] = normal(L, N, r, std=0.02)
    s["scale"] = 0.5 + 1.5 * torch.rand(L, generator=g, device=dev)
    s["ids"] = _rows_to_adapters(g, M, L, case["order"])
    if case["train"]:
        s["dy"] = normal(M, N, std=0.01)
        for n in ("x", "a", "b"):
            s[n].requires_grad_(True)
    return s


# ----------------------------------------------------------------- plain forms --
def _route(s):
    z = s["x"].double() @ s["router_w"].double().t()
    if s["router_b"] is not None:
        z = z + s["router_b"].double()
    p = (z - z.amax(dim=1, keepdim=True)).exp()
    p = p / p.sum(dim=1, keepdim=True)
    idx = z.sort(dim=1, descending=True, stable=True).indices[:, :s["k"]]
    w = p.gather(1, idx)
    if s["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    return idx, w.float()


def _few_plain(s):
    idx, w = (s["idx"], s["w"]) if s["given"] else _route(s)
    T, E = s["T"], s["E"]
    gate = torch.zeros(T, E + 1, device=w.device)
    gate = gate.scatter_add(1, torch.where(idx >= 0, idx, E), w)[:, :E]
    a = torch.matmul(s["x"].float(), s["w1"].float().transpose(1, 2))  # [E, T, F]
    h = 0.5 * a * (1.0 + torch.erf(a * math.sqrt(0.5)))
    y = torch.bmm(h, s["w2"].float().transpose(1, 2))  # [E, T, H]
    out = (y * gate.t()[:, :, None]).sum(dim=0).to(s["x"].dtype)
    return out if s["given"] else (out, idx, w)


def _lora_plain(s):
    x, w, a, b = (s[n].detach().float() for n in ("x", "weight", "a", "b"))
    L, r, K = a.shape
    ids = s["ids"]
    own_columns = ids[:, None] == torch.arange(L, device=ids.device)[None, :]
    mask = (own_columns * s["scale"]).repeat_interleave(r, dim=1)  # [M, L r]
    a_all, b_all = a.reshape(L * r, K), b.transpose(1, 2).reshape(L * r, -1)
    sm = (x @ a_all.t()) * mask
    dt = s["x"].dtype
    y = (x @ w.t() + sm @ b_all).to(dt)
    if not s["train"]:
        return y
    dy = s["dy"].float()
    tm = (dy @ b_all.t()) * mask
    dx = dy @ w + tm @ a_all
    da = (tm.t() @ x).reshape(L, r, K)
    db = (sm.t() @ dy).reshape(L, r, -1).transpose(1, 2)
    return y, dx.to(dt), da.to(dt), db.to(dt).contiguous()


def run(state):
    s = state
    if not own:
        return _few_plain(s) if s["kind"] == "few" else _lora_plain(s)
    import moe_overlap_b200 as mo

    if s["kind"] == "few":
        if s["given"]:
            return mo.experts_few_tokens(s["x"], s["w1"], s["w2"], s["idx"], s["w"])
        return mo.moe_few_tokens(s["x"], s["router_w"], s["w1"], s["w2"], s["k"],
                                 router_bias=s["router_b"], renormalize=s["renorm"])
    y = mo.lora_linear(s["x"], s["weight"], s["a"], s["b"], s["ids"], scale=s["scale"])
    if not s["train"]:
        return y
    dx, da, db = torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["dy"])
    return y.detach(), dx, da, db


# ------------------------------------------------------------------------ work --
def work(case):
    if case["kind"] == "few":
        T, E, H, F, k = (case[n] for n in ("T", "E", "H", "F", "k"))
        rows = (T - T // 4 if case["given"] else T)
        touched = E * (1.0 - (1.0 - k / E) ** rows)  # experts that some token takes, expected
        nbytes = touched * 2 * H * F * 2 + 2 * T * H * 2 + T * k * 12
        flops = rows * k * 4.0 * H * F
        if not case["given"]:
            nbytes += E * H * 2
            flops += 2.0 * T * E * H
        return {"bytes": nbytes, "flops": flops}
    M, K, N, L, r = (case[n] for n in ("M", "K", "N", "L", "r"))
    used = L * (1.0 - (1.0 - 0.875 / L) ** M)
    adapters = used * r * (K + N) * 2
    nbytes = (M * K + N * K + M * N) * 2 + adapters + M * 8
    flops = 2.0 * M * K * N + 2.0 * M * r * (K + N) * 0.875
    if case["train"]:  # dy and the weight read, dx written, x read again, both gradients written
        nbytes += (M * N + N * K + 2 * M * K) * 2 + adapters + L * r * (K + N) * 2
        flops += 2.0 * M * K * N + 4.0 * M * r * (K + N) * 0.875
    return {"bytes": nbytes, "flops": flops}


# ----------------------------------------------------------------- in 64 bits --
def _few_exact(s):
    x = s["x"].double()
    T, k = s["T"], s["k"]
    if s["given"]:
        idx, w = s["idx"], s["w"].double()
    else:
        z = torch.stack([(x * row).sum(dim=1) for row in s["router_w"].double()], dim=1)
        if s["router_b"] is not None:
            z = z + s["router_b"].double()
        logp = z - torch.logsumexp(z, dim=1, keepdim=True)
        idx = torch.stack([torch.tensor(sorted(range(s["E"]), key=lambda e: (-row[e], e))[:k])
                           for row in z.tolist()]).to(x.device)
        logw = logp.gather(1, idx)
        w = torch.softmax(logw, dim=1) if s["renorm"] else logw.exp()
    out = torch.zeros_like(x)
    for e in range(s["E"]):
        t, j = (idx == e).nonzero(as_tuple=True)
        if t.numel():
            a = x[t] @ s["w1"][e].double().t()
            h = a * 0.5 * torch.special.erfc(-a / math.sqrt(2.0))
            out.index_add_(0, t, (h @ s["w2"][e].double().t()) * w[t, j][:, None])
    return out if s["given"] else (out, idx, w)


def _lora_exact(s):
    x, weight, dy = s["x"].detach().double(), s["weight"].double(), s.get("dy")
    y = x @ weight.t()
    if s["train"]:
        dy = dy.double()
        dx = dy @ weight
        da, db = torch.zeros_like(s["a"], dtype=torch.float64), torch.zeros_like(s["b"], dtype=torch.float64)
    for i in range(s["L"]):
        rows = (s["ids"] == i).nonzero()[:, 0]
        a, b, c = s["a"][i].detach().double(), s["b"][i].detach().double(), s["scale"][i].double()
        low = c * (x[rows] @ a.t())
        y[rows] += low @ b.t()
        if s["train"]:
            back = c * (dy[rows] @ b)
            dx[rows] += back @ a
            da[i], db[i] = back.t() @ x[rows], dy[rows].t() @ low
    return (y, dx, da, db) if s["train"] else y


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _few_exact(s) if s["kind"] == "few" else _lora_exact(s)
