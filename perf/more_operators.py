"""The operators with which a hybrid language model ends a training step and
answers in 8 bits, as a program calls them: the cross entropy of a linear head
over a large vocabulary, the e4m3 product with scales of 128 columns, and the
e4m3 key and value cache.

Kinds of call:
  xent_fwd     linear_xent: the losses of given rows (scoring)
  xent_train   linear_xent and linear_xent_bwd
  fp8_linear   fp8_linear on rows that are in 8 bits already (as the norm leaves them)
  fp8_mixer    quantize_fp8 of 16-bit rows (as a mixer leaves them), then fp8_linear
  cache_step   cache_write_fp8 of the new tokens, then window_attn_decode_fp8
  cache_write  cache_write_fp8 of whole prompts
  cache_read   cache_read_fp8: rows of a cache in 16 bits again

With `own` false, run() computes them in elementary torch operations in 32
bits; with `own` true it calls the package.
"""

import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0    # largest finite value of e4m3
DEV = "cuda"


def _package():
    import importlib
    return importlib.import_module("v100-attention-lab_amd")


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # scoring the last rows of a few sequences over a vocabulary that no tile divides
        {"name": "xent_score_bf16", "kind": "xent_fwd", "N": 48, "D": 2048, "V": 50257, "dtype": "bf16", "ignored": 0.0},
        # a training step of a small model on ragged rows, a tenth of them padding
        {"name": "xent_train_f16_odd", "kind": "xent_train", "N": 1111, "D": 1096, "V": 10007, "dtype": "f16",
         "ignored": 0.1},
        # a training step at the benchmark's headline rows (2 x 4096, 16 heads of 128)
        {"name": "xent_train_bf16", "kind": "xent_train", "N": 8192, "D": 2048, "V": 32000, "dtype": "bf16",
         "ignored": 0.0},
        # the same rows of a wider model with a large vocabulary
        {"name": "xent_train_large", "kind": "xent_train", "N": 8192, "D": 4096, "V": 128000, "dtype": "bf16",
         "ignored": 0.05},
        # one sequence answering: latency
        {"name": "fp8_one", "kind": "fp8_linear", "M": 1, "K": 2048, "N": 2048, "group": 128, "out": "bf16"},
        # a decode step of 16 sequences: the delta rule's input product (16 heads of 3 * 128 + 2)
        {"name": "fp8_step", "kind": "fp8_linear", "M": 16, "K": 2048, "N": 6176, "group": 128, "out": "bf16"},
        # a ragged prompt through an output product, the rows quantised on the way
        {"name": "fp8_mixer_ragged", "kind": "fp8_mixer", "M": 777, "K": 2048, "N": 2048, "group": 128, "out": "f16"},
        # a prefill of 8192 rows
        {"name": "fp8_prefill", "kind": "fp8_linear", "M": 8192, "K": 4096, "N": 8192, "group": 128, "out": "bf16"},
        # one sequence far into a long cache, every key visible: latency
        {"name": "cache_step_one", "kind": "cache_step", "B": 1, "T": 1, "S": 65536, "Hq": 16, "Hk": 4, "D": 128,
         "dtype": "bf16", "window": 0, "sinks": 0, "ragged": False},
        # a serving batch of 32 sequences of different lengths
        {"name": "cache_step_batch", "kind": "cache_step", "B": 32, "T": 1, "S": 16384, "Hq": 16, "Hk": 4, "D": 128,
         "dtype": "bf16", "window": 4096, "sinks": 4, "ragged": True},
        # the prompts of 8 sequences into their caches
        {"name": "cache_write_prompts", "kind": "cache_write", "B": 8, "T": 2048, "S": 4096, "Hq": 16, "Hk": 4,
         "D": 128, "dtype": "bf16"},
        # a cache of 8 sequences read back, for a prefill that continues them
        {"name": "cache_read_back", "kind": "cache_read", "B": 8, "S": 4096, "Hk": 4, "D": 128, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the ranges above: 1 to 65536 rows (odd ones mostly), any
    vocabulary, head sizes 64 and 128, 1 to 4 query heads for each key head,
    at most the work of the largest listed case."""
    kind = rng.choice(["xent_fwd", "xent_train", "xent_train", "fp8_linear", "fp8_linear", "fp8_mixer", "cache_step",
                       "cache_step", "cache_write", "cache_read"])
    if kind.startswith("xent"):
        D = rng.choice([64, 256, 2048, 4096, 8 * _log(rng, 8, 512)])
        V = rng.choice([32000, 128000, _log(rng, 60, 128000)])
        N = _log(rng, 1, min(32768, 4_000_000_000_000 // (D * V), 1_500_000_000 // V))
        return {"kind": kind, "N": N, "D": D, "V": V, "dtype": rng.choice(["f16", "bf16", "bf16"]),
                "ignored": rng.choice([0.0, 0.05, 0.5])}
    if kind.startswith("fp8"):
        K = 128 * _log(rng, 1, 64)
        N = rng.choice([128 * _log(rng, 1, 64), _log(rng, 1, 16384)])
        M = _log(rng, 1, min(65536, 270_000_000_000 // (N * K), 130_000_000 // max(N, K)))
        return {"kind": kind, "M": M, "K": K, "N": N, "group": rng.choice([0, 128, 128]),
                "out": rng.choice(["bf16", "bf16", "f16", "f32"])}
    D = rng.choice([64, 128])
    Hk = rng.choice([1, 2, 4, 8])
    Hq = Hk * rng.choice([1, 2, 3, 4])
    dtype = rng.choice(["f16", "bf16"])
    S = _log(rng, 16, 65536)
    B = _log(rng, 1, max(1, min(64, 100_000_000 // (S * Hk * D))))
    if kind == "cache_read":
        return {"kind": kind, "B": B, "S": S, "Hk": Hk, "D": D, "dtype": dtype}
    case = {"kind": kind, "B": B, "S": S, "Hq": Hq, "Hk": Hk, "D": D, "dtype": dtype}
    if kind == "cache_write":
        return dict(case, T=_log(rng, 1, min(S, max(1, 134_000_000 // (B * (Hq + 2 * Hk) * D)))))
    # every key visible only where all of them are a fair amount of work
    window = 0 if rng.random() < 0.3 and B * S <= 131072 else _log(rng, 16, 4096)
    return dict(case, T=rng.choice([1, 1, 1, 2, 4]), window=window, sinks=rng.choice([0, 1, 4, 16, 100]),
                ragged=rng.random() < 0.7)


def _cache_lens(case, seed):
    """Keys of each sequence of a call, the new tokens among them."""
    T, S = case["T"], case["S"]
    if case["kind"] == "cache_write":
        return [S - (S - T) // 3] * case["B"]
    if not case["ragged"]:
        return [max(T, S - S // 13)] * case["B"]
    r = torch.Generator().manual_seed(seed)
    lo = min(T, S)
    return (lo + torch.randint(0, S - lo + 1, (case["B"],), generator=r)).tolist()


def _to_fp8(x, scale):
    """x over its scale (of zero: zeros), rounded to e4m3."""
    return torch.clamp(torch.where(scale > 0, x / scale, 0.0), -FP8_MAX, FP8_MAX).to(FP8)


def _quant_rows(x, group):
    """[M, K] in groups of columns: the bytes [M, K] and the scales [M, K / group]."""
    g = x.float().unflatten(-1, (-1, group))
    scale = g.abs().amax(-1, keepdim=True) / FP8_MAX
    return _to_fp8(g, scale).flatten(-2), scale.squeeze(-1)


def _quant_weight(w):
    """[N, K] in blocks of 128 x 128: the bytes [N, K] and the scales."""
    N, K = w.shape
    blocks = torch.nn.functional.pad(w.float(), (0, 0, 0, -N % 128)).view(-1, 128, K // 128, 128)
    scale = blocks.abs().amax((1, 3), keepdim=True) / FP8_MAX
    return _to_fp8(blocks, scale).view(-1, K)[:N].contiguous(), scale[:, 0, :, 0].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    kind = case["kind"]
    st = {"kind": kind, "case": case}
    if kind.startswith("xent"):
        N, D, V, dt = case["N"], case["D"], case["V"], DTYPES[case["dtype"]]
        # rows as the last norm leaves them; logits of a standard deviation of 2
        st["x"] = rn(N, D).to(dt)
        st["w"] = (rn(V, D) * (2.0 / D ** 0.5)).to(dt)
        target = torch.randint(0, V, (N,), generator=gen, device=DEV)
        out = torch.rand(N, generator=gen, device=DEV) < case["ignored"]
        st["target"] = torch.where(out, -100, target)
        if kind == "xent_train":
            # the gradient of a mean with a weight for each row
            st["dloss"] = (0.5 + torch.rand(N, generator=gen, device=DEV)) / N
    elif kind.startswith("fp8"):
        M, K, N = case["M"], case["K"], case["N"]
        x = rn(M, K) * (1.0 + 7.0 * (torch.rand(K, generator=gen, device=DEV) < 0.01))
        st["w"], st["ws"] = _quant_weight(rn(N, K) * K ** -0.5)
        st["out"] = DTYPES[case["out"]]
        if kind == "fp8_mixer":
            st["x"] = x.to(torch.float32 if case["out"] == "f32" else st["out"])
        else:
            st["x"], st["xs"] = _quant_rows(x, case["group"] or K)
    else:
        B, S, Hk, D, dt = (case[n] for n in ("B", "S", "Hk", "D", "dtype"))
        # rows of different sizes, as keys without a norm have them
        size = lambda *s: torch.exp(0.5 * rn(*s, 1))
        for n in ("k", "v"):
            st[n + "c"], scale = _quant_rows(rn(B * S * Hk, D) * size(B * S * Hk), D)
            st[n + "c"] = st[n + "c"].view(B, S, Hk, D)
            st[n + "s"] = scale.view(B, S, Hk).contiguous()
        st["dtype"] = DTYPES[dt]
        if kind != "cache_read":
            T, Hq = case["T"], case["Hq"]
            # q, k and v as one product's output gives them
            qkv = (rn(B, T, Hq + 2 * Hk, D) * size(B, T, Hq + 2 * Hk)).to(st["dtype"])
            st["q"], st["k"], st["v"] = qkv.split([Hq, Hk, Hk], 2)
            st["lens"] = torch.tensor(_cache_lens(case, seed), dtype=torch.int32, device=DEV)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    if own:
        return _run_own(st, st["case"])
    kind = st["kind"]
    if kind.startswith("xent"):
        return _plain_xent(st)
    if kind.startswith("fp8"):
        return _plain_fp8(st, st["case"])
    if kind == "cache_read":
        return {"k": _values(st["kc"], st["ks"]).to(st["dtype"]), "v": _values(st["vc"], st["vs"]).to(st["dtype"])}
    _plain_write(st, st["case"])
    out = {n: st[n] for n in ("kc", "vc", "ks", "vs")}
    if kind == "cache_step":
        out["o"] = _plain_decode(st, st["case"])
    return out


def _run_own(st, case):
    gdn, kind = _package(), st["kind"]
    if kind == "xent_fwd":
        loss, lse = gdn.linear_xent(st["x"], st["w"], st["target"], return_lse=True)
        return {"loss": loss, "lse": lse}
    if kind == "xent_train":
        loss, lse = gdn.linear_xent(st["x"], st["w"], st["target"], return_lse=True)
        dx, dw = gdn.linear_xent_bwd(st["x"], st["w"], st["target"], lse, st["dloss"])
        return {"loss": loss, "lse": lse, "dx": dx, "dw": dw}
    if kind == "fp8_linear":
        return {"y": gdn.fp8_linear(st["x"], st["xs"], st["w"], st["ws"], out_dtype=st["out"])}
    if kind == "fp8_mixer":
        x, xs = gdn.quantize_fp8(st["x"], group=case["group"] or None)
        return {"x": x, "xs": xs, "y": gdn.fp8_linear(x, xs, st["w"], st["ws"], out_dtype=st["out"])}
    if kind == "cache_read":
        k, v = gdn.cache_read_fp8(st["kc"], st["vc"], st["ks"], st["vs"], dtype=st["dtype"])
        return {"k": k, "v": v}
    gdn.cache_write_fp8(st["k"], st["v"], st["kc"], st["vc"], st["ks"], st["vs"], st["lens"])
    out = {n: st[n] for n in ("kc", "vc", "ks", "vs")}
    if kind == "cache_step":
        out["o"] = gdn.window_attn_decode_fp8(st["q"], st["kc"], st["vc"], st["ks"], st["vs"], st["lens"],
                                              case["window"] or None, case["sinks"])
    return out


# ---------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits, rounded once at the end
# ---------------------------------------------------------------------------

def _plain_xent(st):
    x, w, target = st["x"].float(), st["w"].float(), st["target"]
    counts = (target >= 0) & (target < w.shape[0])
    at = torch.where(counts, target, 0)[:, None]
    logits = x @ w.T
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - top)
    s = p.sum(-1, keepdim=True)
    lse = (top + torch.log(s)).squeeze(1)
    out = {"loss": torch.where(counts, lse - logits.gather(1, at).squeeze(1), 0.0), "lse": torch.where(counts, lse, 0.0)}
    if st["kind"] == "xent_fwd":
        return out
    p.div_(s)
    p.scatter_add_(1, at, torch.full_like(p[:, :1], -1.0))
    p.mul_(torch.where(counts, st["dloss"], 0.0)[:, None])
    out["dx"] = (p @ w).to(st["x"].dtype)
    out["dw"] = (p.T @ x).to(st["w"].dtype)
    return out


def _values(q, scale):
    """What bytes and the scales of their last dimension's groups stand for."""
    return (q.float().unflatten(-1, (scale.shape[-1], -1)) * scale[..., None]).flatten(-2) if scale.dim() == q.dim() \
        else q.float() * scale[..., None]


def _plain_fp8(st, case):
    out = {}
    x, xs = st["x"], st.get("xs")
    if st["kind"] == "fp8_mixer":
        x, xs = _quant_rows(x, case["group"] or case["K"])
        out = {"x": x, "xs": xs}
    w = _values(st["w"], st["ws"].repeat_interleave(128, 0)[:case["N"]])
    out["y"] = (_values(x, xs) @ w.T).to(st["out"])
    return out


def _plain_write(st, case):
    B, T = case["B"], case["T"]
    rows = st["lens"].long()[:, None] - T + torch.arange(T, device=DEV)      # (none of them before the first)
    which = torch.arange(B, device=DEV)[:, None]
    for n in ("k", "v"):
        q, scale = _quant_rows(st[n], case["D"])
        st[n + "c"].view(torch.uint8)[which, rows] = q.view(torch.uint8)
        st[n + "s"][which, rows] = scale.squeeze(-1)


def _plain_decode(st, case):
    B, T, S, Hq, Hk, D = (case[n] for n in ("B", "T", "S", "Hq", "Hk", "D"))
    W, G, scale = min(case["window"] or S, S), Hq // Hk, D ** -0.5
    n = st["lens"].long()
    win = (n - T - (W - 1))[:, None] + torch.arange(W - 1 + T, device=DEV)
    sink = torch.arange(min(case["sinks"], S), device=DEV).expand(B, -1)
    at = torch.clamp(torch.cat([win, sink], 1), 0, S - 1)              # [B, L]
    i = (n[:, None] - T + torch.arange(T, device=DEV))[:, :, None]     # [B, T, 1]
    seen_w = (win[:, None] >= 0) & (win[:, None] <= i) & (win[:, None] > i - W)
    seen = torch.cat([seen_w, sink[:, None] <= i - W], 2)
    which = torch.arange(B, device=DEV)[:, None]
    k, v = (_values(st[c + "c"].view(torch.uint8)[which, at].view(FP8), st[c + "s"][which, at])
            .permute(0, 2, 1, 3).contiguous() for c in ("k", "v"))
    q = st["q"].float().reshape(B, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * T, D)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, Hk, G, T, -1) * scale
    s = torch.where(seen[:, None, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
    p = p / torch.clamp(p.sum(-1, keepdim=True), min=1e-38)
    o = torch.matmul(p.view(B, Hk, G * T, -1), v).view(B, Hk, G, T, D)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(st["q"].dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    kind = case["kind"]
    if kind.startswith("xent"):
        N, D, V, es = case["N"], case["D"], case["V"], _size(case["dtype"])
        counted = N * (1.0 - case["ignored"])
        if kind == "xent_fwd":
            return {"bytes": es * (N + V) * D + 16 * N, "flops": 2 * counted * D * V}
        # rows and weights in, their gradients out; the logits' product and one for each gradient
        return {"bytes": 2 * es * (N + V) * D + 20 * N, "flops": 6 * counted * D * V}
    if kind.startswith("fp8"):
        M, K, N = case["M"], case["K"], case["N"]
        groups = K // (case["group"] or K)
        by = M * K + 4 * M * groups + N * K + 4 * -(-N // 128) * (K // 128) + M * N * _size(case["out"])
        if kind == "fp8_mixer":
            by += M * K * _size(case["out"])
        return {"bytes": by, "flops": 2 * M * K * N}
    B, S, Hk, D, es = case["B"], case["S"], case["Hk"], case["D"], _size(case["dtype"])
    if kind == "cache_read":
        return {"bytes": 2 * B * S * Hk * (D * (1 + es) + 4), "flops": 2 * B * S * Hk * D}
    T, new = case["T"], 2 * B * case["T"] * Hk
    by = new * (D * (1 + es) + 4)
    if kind == "cache_write":
        return {"bytes": by, "flops": 3 * new * D}
    W, sinks = case["window"] or S, case["sinks"]
    lens = [max(T, S - S // 13) if not case["ragged"] else (T + S) // 2] * B
    keys = sum(min(n, W + T - 1) + min(sinks, max(n - W, 0)) for n in lens)
    return {"bytes": by + 2 * keys * Hk * (D + 4) + 2 * es * B * T * case["Hq"] * D,
            "flops": 4 * D * case["Hq"] * T * keys}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind.startswith("xent"):
        return _exact_xent(st, case)
    if kind.startswith("fp8"):
        return _exact_fp8(st, case)
    if kind == "cache_read":
        return {n: st[n + "c"].double() * st[n + "s"].double()[..., None] for n in ("k", "v")}
    return _exact_cache(st, case)


def _exact_xent(st, case):
    """1024 rows at a time."""
    N, V = case["N"], case["V"]
    train = case["kind"] == "xent_train"
    w = st["w"].double()
    out = {"loss": [], "lse": [], "dx": []}
    dw = torch.zeros_like(w) if train else None
    for r0 in range(0, N, 1024):
        x, t = st["x"][r0:r0 + 1024].double(), st["target"][r0:r0 + 1024]
        rows = torch.arange(t.numel(), device=DEV)
        counts = (t >= 0) & (t < V)
        l = torch.mm(x, w.t())
        lse = torch.logsumexp(l, 1)
        t = torch.where(counts, t, 0)
        out["loss"].append(torch.where(counts, lse - l[rows, t], 0.0))
        out["lse"].append(torch.where(counts, lse, 0.0))
        if train:
            g = torch.exp(l - lse[:, None])
            g[rows, t] -= 1.0
            g *= torch.where(counts, st["dloss"][r0:r0 + 1024].double(), 0.0)[:, None]
            out["dx"].append(torch.mm(g, w))
            dw += torch.mm(g.t(), x)
    out = {n: torch.cat(v) for n, v in out.items() if v}
    return dict(out, dw=dw) if train else out


def _round_e4m3(x):
    """To 3 bits behind the leading one, not below 2^-9; halves to even."""
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(x.abs(), min=1e-30))), min=-6.0) - 3.0)
    return torch.clamp(torch.round(x / step) * step, -FP8_MAX, FP8_MAX)


def _exact_quant(x, group):
    g = x.double().unflatten(-1, (-1, group))
    scale = g.abs().amax(-1, keepdim=True) / FP8_MAX
    return _round_e4m3(torch.where(scale > 0, g / scale, 0.0)).flatten(-2), scale.squeeze(-1)


def _exact_fp8(st, case):
    K, N = case["K"], case["N"]
    out = {}
    if case["kind"] == "fp8_mixer":
        x, xs = _exact_quant(st["x"], case["group"] or K)
        out = {"x": x, "xs": xs}
    else:
        x, xs = st["x"].double(), st["xs"].double()
    x = x * xs.repeat_interleave(K // xs.shape[1], 1)
    block = torch.arange(N, device=DEV) // 128
    w = st["w"].double() * st["ws"].double()[block].repeat_interleave(128, 1)
    return dict(out, y=torch.mm(x, w.t()))


def _exact_cache(st, case):
    B, T, S, D = case["B"], case["T"], case["S"], case["D"]
    lens = st["lens"].tolist()
    out = {}
    for n in ("k", "v"):
        q, scale = _exact_quant(st[n], D)
        c, s = st[n + "c"].to(torch.float32), st[n + "s"].double()
        for b in range(B):
            c[b, lens[b] - T:lens[b]] = q[b].float()
            s[b, lens[b] - T:lens[b]] = scale[b, ..., 0]
        out[n + "c"], out[n + "s"] = c, s
    if case["kind"] == "cache_write":
        return out
    Hq, Hk = case["Hq"], case["Hk"]
    G, W = Hq // Hk, case["window"] or S
    o = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=DEV)
    for b in range(B):
        j = torch.arange(lens[b], device=DEV)
        for t in range(T):
            i = lens[b] - T + t
            see = j[(j <= i) & ((j > i - W) | (j < case["sinks"]))]
            K, V = (out[n + "c"][b, see].double() * out[n + "s"][b, see][..., None] for n in ("k", "v"))
            for h in range(Hq):
                p = torch.softmax(torch.mv(K[:, h // G], st["q"][b, t, h].double()) * D ** -0.5, 0)
                o[b, t, h] = torch.mv(V[:, h // G].t(), p)
    return dict(out, o=o)
