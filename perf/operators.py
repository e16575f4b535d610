"""Cases of the operators for long texts: attention in a sliding window with
sinks (training and single tokens), dropout with the residual sum, and the log
probabilities of given tokens.

Each case names its operator in "op":

  attention  forward and backward over packed q | k | v rows; `lengths` says
             how the sequences' lengths are drawn ("full": all S, "ragged":
             anything from 0 to S, one of them 0 when there are several)
  step       one new token a sequence against a key-value ring; its row of the
             ring is written too, so the ring comes back with the result
  logprobs   log probability, entropy and top alternatives of T rows of V
             logits; with `grad` the gradient of a weighted sum of the log
             probabilities and entropies as well
  dropout    residual + dropout(x), and the gradient of x
"""

import math

import torch

own = False

DEV = "cuda"
LOG2E = math.log2(math.e)
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # the smallest training call: a short text through a four-head model
        dict(name="attention short text", op="attention", B=1, S=77, H=4, Hkv=2, hd=64, window=32,
             sinks=4, lengths="full"),
        # a microbatch of the 12 x 128-head GPT, half of its keys out of the window
        dict(name="attention 12 heads", op="attention", B=4, S=2048, H=12, Hkv=12, hd=128,
             window=512, sinks=0, lengths="full"),
        # padded texts of an odd longest length on 80-wide heads, one of them empty
        dict(name="attention ragged, hd 80", op="attention", B=3, S=1999, H=32, Hkv=32, hd=80,
             window=640, sinks=16, lengths="ragged"),
        # a long text on grouped heads: what the window is for
        dict(name="attention long text", op="attention", B=1, S=8192, H=32, Hkv=8, hd=128,
             window=1024, sinks=4, lengths="full"),
        # one answer, token by token, far past the ring's end
        dict(name="step one answer", op="step", B=1, H=32, Hkv=8, hd=128, window=1024, sinks=4,
             cap=1028, longest=20000),
        # a batch of answers of every age, some of them over
        dict(name="step batch, hd 64", op="step", B=48, H=32, Hkv=8, hd=64, window=2047, sinks=16,
             cap=2064, longest=6000),
        # every head with keys of its own, a wide window in a cache that never wraps
        dict(name="step wide window", op="step", B=8, H=40, Hkv=40, hd=128, window=4096, sinks=64,
             cap=6000, longest=6000),
        # one sampled token: its log probability and 20 alternatives
        dict(name="logprobs one token", op="logprobs", T=1, V=128256, ld=128256, dtype="bf16",
             top=20, masked=0.0, grad=False),
        # scoring under a vocabulary mask, rows padded apart
        dict(name="logprobs masked", op="logprobs", T=1000, V=32768, ld=32776, dtype="bf16", top=5,
             masked=0.6, grad=False),
        # an update from log probabilities and entropies; odd vocabulary, fp32 logits
        dict(name="logprobs training", op="logprobs", T=4096, V=50257, ld=50257, dtype="fp32",
             top=0, masked=0.0, grad=True),
        # the smallest residual branch
        dict(name="dropout small", op="dropout", rows=512, d=768, dtype="bf16", p=0.1, resid=True),
        # the residual branch of a long microbatch of the 5120-wide model
        dict(name="dropout large", op="dropout", rows=16384, d=5120, dtype="bf16", p=0.1,
             resid=True),
    ]


def _log_int(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.01)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "step", "step", "logprobs", "logprobs", "dropout"])
    if op == "attention":
        S = _log_int(rng, 1, 8192)
        H, Hkv = rng.choice([(4, 2), (12, 12), (16, 4), (25, 25), (32, 8), (32, 32), (6, 1)])
        most = max(1, int(32 * 8192 * 8192 / (S * S * H)))
        return dict(op=op, B=min(_log_int(rng, 1, 16), most), S=S, H=H, Hkv=Hkv,
                    hd=rng.choice([64, 80, 96, 128]), window=_log_int(rng, 1, max(2, S + S // 4)),
                    sinks=rng.choice([0, 1, 4, 64, 200]), lengths=rng.choice(["full", "ragged"]))
    if op == "step":
        H, Hkv = rng.choice([(4, 2), (12, 12), (16, 4), (32, 8), (40, 40), (6, 1)])
        hd, sinks = rng.choice([64, 80, 96, 128]), rng.choice([0, 1, 4, 64])
        window = _log_int(rng, 1, 8192)
        cap = sinks + window + rng.choice([0, 0, 1, 77, 1000])
        most = max(1, int(8 * 6000 * 40 * 128 / (cap * Hkv * hd)))
        return dict(op=op, B=min(_log_int(rng, 1, 128), most), H=H, Hkv=Hkv, hd=hd, window=window,
                    sinks=sinks, cap=cap, longest=_log_int(rng, 1, 4 * cap))
    if op == "logprobs":
        V = _log_int(rng, 200, 200000)
        ld = V + rng.choice([0, 0, 1, 8, 40])
        dtype, top = rng.choice(["bf16", "fp32"]), rng.choice([0, 1, 5, 20, 32])
        return dict(op=op, T=_log_int(rng, 1, max(1, min(6000, 4096 * 50257 // ld))), V=V, ld=ld,
                    dtype=dtype, top=top, masked=rng.choice([0.0, 0.0, 0.5, 0.99]),
                    grad=rng.choice([True, False]))
    d = _log_int(rng, 1, 8192)
    return dict(op=op, rows=_log_int(rng, 1, max(1, 16384 * 2048 // d)), d=d,
                dtype=rng.choice(["bf16", "bf16", "fp32"]), p=rng.choice([0.0, 0.05, 0.1, 0.5]),
                resid=rng.choice([True, False]))


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1 + int(seed))
    return g


def _normal(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _lengths(c, g):
    if c["lengths"] == "full":
        return None
    n = torch.randint(0, c["S"] + 1, (c["B"],), generator=g, device=DEV)
    if c["B"] > 1:
        n[c["B"] - 1] = 0
        n[0] = c["S"]
    return n.to(torch.int32)


def prepare(case, seed):
    c, g = case, _gen(seed)
    op = c["op"]
    if op == "attention":
        rows, width = c["B"] * c["S"], (c["H"] + 2 * c["Hkv"]) * c["hd"]
        # projections of a normalised stream: unit variance; gradients are small
        return dict(c=c, qkv=_normal(g, rows, width),
                    dout=_normal(g, rows, c["H"] * c["hd"], scale=0.02), lengths=_lengths(c, g))
    if op == "step":
        width = 2 * c["Hkv"] * c["hd"]
        # the number of tokens that each answer has so far; every seventh is over
        pos = torch.randint(0, c["longest"], (c["B"],), generator=g, device=DEV)
        pos = torch.where(torch.arange(c["B"], device=DEV) % 7 == 6, -1, pos)
        return dict(c=c, qkv=_normal(g, c["B"], c["H"] * c["hd"] + width),
                    cache=_normal(g, c["B"], c["cap"], width), pos=pos)
    if op == "logprobs":
        T, V, ld = c["T"], c["V"], c["ld"]
        # a few tokens stand out of each row, as they do in a trained model's
        x = torch.randn(T, ld, generator=g, device=DEV)
        x = (x * 1.5 + 9.0 * (x > 3.0)).to(DT[c["dtype"]])
        if c["masked"]:
            x.masked_fill_(torch.rand(1, ld, generator=g, device=DEV) < c["masked"], -math.inf)
        targets = torch.randint(0, V, (T,), generator=g, device=DEV)
        # prompt rows have no given token
        targets = torch.where(torch.rand(T, generator=g, device=DEV) < 0.1, -1, targets)
        if c["masked"]:  # nobody is given a token that cannot come
            targets = torch.where(x[:, :V].gather(1, targets.clamp(min=0)[:, None])[:, 0] == -math.inf,
                                  -1, targets)
        return dict(c=c, logits=x, targets=targets,
                    g_logp=_normal(g, T, scale=1.0 / T, dtype=torch.float32),
                    g_entropy=_normal(g, T, scale=0.1 / T, dtype=torch.float32))
    dt = DT[c["dtype"]]
    return dict(c=c, x=_normal(g, c["rows"], c["d"], dtype=dt),
                resid=_normal(g, c["rows"], c["d"], dtype=dt) if c["resid"] else None,
                dy=_normal(g, c["rows"], c["d"], scale=0.02, dtype=dt),
                seed=(int(seed) * 2654435761 + 12345) & ((1 << 62) - 1), stream=(7 << 33) + int(seed))


# ----------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _run_own(s)
    return {"attention": _attention, "step": _step, "logprobs": _logprobs,
            "dropout": _dropout}[s["c"]["op"]](s)


def _run_own(s):
    from elysium_wan_b200 import ops

    c = s["c"]
    if c["op"] == "attention":
        shape = (c["B"], c["S"], c["H"], c["hd"], c["Hkv"])
        mask = dict(window=c["window"], sinks=c["sinks"], lengths=s["lengths"])
        o, lse = ops.window_attention_fwd(s["qkv"], *shape, **mask)
        dqkv = ops.window_attention_bwd(s["qkv"], o, s["dout"], lse, *shape, **mask)
        return {"o": o, "lse": lse, "dqkv": dqkv}
    if c["op"] == "step":
        o = ops.window_attention_step(s["qkv"], s["cache"], s["pos"], c["H"], c["hd"], c["Hkv"],
                                      window=c["window"], sinks=c["sinks"])
        return {"o": o, "cache": s["cache"]}
    if c["op"] == "logprobs":
        r = ops.token_logprobs(s["logits"], c["V"], s["targets"], top=c["top"])
        out = {"logp": r.logp, "entropy": r.entropy, "lse": r.lse}
        if c["top"]:
            out.update(top_logp=r.top_logp, top_ids=r.top_ids)
        if c["grad"]:
            out["dlogits"] = ops.token_logprobs_bwd(s["logits"], c["V"], s["targets"], r.lse,
                                                    r.entropy, s["g_logp"], s["g_entropy"],
                                                    ld_grad=c["V"])
        return out
    y = ops.dropout_add(s["x"], s["resid"], c["p"], s["seed"], s["stream"])
    return {"y": y, "dx": ops.dropout_bwd(s["dy"], c["p"], s["seed"], s["stream"])}


def _split(c, qkv, f):
    """q [B, Hkv, rep, S, hd], k and v [B, Hkv, 1, S, hd] of packed rows."""
    B, S, H, Hkv, hd = c["B"], c["S"], c["H"], c["Hkv"], c["hd"]
    x = qkv.to(f).view(B, S, H + 2 * Hkv, hd).transpose(1, 2)
    return (x[:, :H].reshape(B, Hkv, H // Hkv, S, hd), x[:, H:H + Hkv, None],
            x[:, H + Hkv:, None])


def _visible(c, lengths):
    i = torch.arange(c["S"], device=DEV)[:, None]
    j = torch.arange(c["S"], device=DEV)[None, :]
    m = (j <= i) & ((i - j < c["window"]) | (j < c["sinks"]))
    if lengths is None:
        return m[None, None, None]
    n = lengths.view(-1, 1, 1, 1, 1)
    return m & (i < n) & (j < n)


def _attention(s):
    c, rows = s["c"], s["c"]["B"] * s["c"]["S"]
    B, S, H, hd = c["B"], c["S"], c["H"], c["hd"]
    q, k, v = _split(c, s["qkv"], torch.float32)
    do = s["dout"].float().view(B, S, H, hd).transpose(1, 2).reshape(q.shape)
    scale = 1.0 / math.sqrt(hd)
    x = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(~_visible(c, s["lengths"]), -math.inf)
    m = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    l = x.sum(-1, keepdim=True)
    p = x.div_(torch.where(l == 0, 1.0, l))
    o = p @ v
    lse = (m + torch.log(l)) * LOG2E
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = do @ v.transpose(-1, -2)
    ds = ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p)
    dq = (ds @ k) * scale
    dk = (ds.transpose(-1, -2) @ q).sum(2) * scale
    flat = lambda t: t.reshape(B, -1, S, hd).transpose(1, 2).reshape(rows, -1)  # noqa: E731
    return {"o": flat(o).to(torch.bfloat16), "lse": lse.view(B, H, S),
            "dqkv": torch.cat([flat(dq), flat(dk), flat(dv)], 1).to(torch.bfloat16)}


def _ring(c, pos):
    """The position that each slot holds once the new tokens are in, and
    whether the new token sees it: [B, cap] both."""
    turn = c["cap"] - c["sinks"]
    slot = torch.arange(c["cap"], device=DEV)[None, :]
    p = pos[:, None]
    last = p - (p - slot) % turn  # the newest position <= pos that slot can hold
    held = torch.where(slot < c["sinks"], slot, last)
    seen = (held <= p) & (held >= torch.where(slot < c["sinks"], 0, c["sinks"]))
    seen &= (p - held < min(c["window"], turn)) | (held < c["sinks"])
    return held, seen & (p >= 0)


def _step(s):
    c, qkv, cache, pos = s["c"], s["qkv"], s["cache"], s["pos"]
    B, H, Hkv, hd = c["B"], c["H"], c["Hkv"], c["hd"]
    turn = c["cap"] - c["sinks"]
    new = torch.where(pos < c["sinks"], pos, c["sinks"] + (pos - c["sinks"]) % turn).clamp(min=0)
    at = torch.arange(B, device=DEV)
    cache[at, new] = torch.where(pos[:, None] >= 0, qkv[:, H * hd:], cache[at, new])
    _, seen = _ring(c, pos)
    q = qkv[:, :H * hd].float().view(B, Hkv, H // Hkv, hd)
    kv = cache.float().view(B, c["cap"], 2, Hkv, hd)
    x = torch.einsum("bgrd,bcgd->bgrc", q, kv[:, :, 0]) / math.sqrt(hd)
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    l = x.sum(-1, keepdim=True)
    o = torch.einsum("bgrc,bcgd->bgrd", x / torch.where(l == 0, 1.0, l), kv[:, :, 1])
    return {"o": o.reshape(B, H * hd).to(torch.bfloat16), "cache": cache}


def _logprobs(s):
    c, t = s["c"], s["targets"]
    x = s["logits"][:, :c["V"]].float()
    m = x.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    # a row without a finite logit gives every token no chance: all logs -inf
    lse = torch.where(z == 0, -math.inf, m + torch.log(z))
    at = torch.where(z == 0, 0.0, lse)
    p = e / torch.where(z == 0, 1.0, z)
    # p log p is 0 where p is
    logp = torch.where(p > 0, x - at, 0.0)
    entropy = -(p * logp).sum(1)
    given = t >= 0
    got = torch.where(given, (x.gather(1, t.clamp(min=0)[:, None]) - at)[:, 0], 0.0)
    out = {"logp": got, "entropy": entropy, "lse": lse[:, 0]}
    if c["top"]:
        v, ids = torch.sort(x, dim=1, descending=True, stable=True)
        out.update(top_logp=v[:, :c["top"]] - at, top_ids=ids[:, :c["top"]].contiguous())
    if c["grad"]:
        gl = torch.where(given, s["g_logp"], 0.0)
        d = -p * (gl[:, None] + s["g_entropy"][:, None] * (logp + entropy[:, None]))
        d.scatter_add_(1, t.clamp(min=0)[:, None], gl[:, None])
        out["dlogits"] = d.to(torch.bfloat16)
    return out


def _words(n, seed, stream):
    """n 32-bit words of the counter-based generator Philox4x32-10 (Salmon et
    al., SC 2011): word e is word e % 4 of the block of counter (e // 4,
    stream) under key seed."""
    low = 0xFFFFFFFF
    blk = torch.arange((n + 3) // 4, device=DEV)
    c = [blk & low, blk >> 32, torch.full_like(blk, stream & low), torch.full_like(blk, stream >> 32)]
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # 64-bit products, modulo 2^64
        c = [((b >> 32) & low) ^ c[1] ^ k0, b & low, ((a >> 32) & low) ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack(c, 1).view(-1)[:n]


def _dropout(s):
    c = s["c"]
    n = c["rows"] * c["d"]
    keep = (_words(n, s["seed"], s["stream"]) >= min(round(c["p"] * 2**32), 2**32 - 1))
    keep = keep.view(c["rows"], c["d"])
    scale = 1.0 / (1.0 - c["p"])
    y = torch.where(keep, s["x"].float() * scale, 0.0)
    if s["resid"] is not None:
        y = y + s["resid"].float()
    return {"y": y.to(s["x"].dtype),
            "dx": torch.where(keep, s["dy"].float() * scale, 0.0).to(s["x"].dtype)}


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "step": _exact_step, "logprobs": _exact_logprobs,
            "dropout": _exact_dropout}[case["op"]](case, s)


def _exact_attention(c, s):
    """Head by head, blocks of queries against the keys they can reach."""
    f = torch.float64
    B, S, H, Hkv, hd = c["B"], c["S"], c["H"], c["Hkv"], c["hd"]
    qkv = s["qkv"].view(B, S, H + 2 * Hkv, hd)
    do = s["dout"].view(B, S, H, hd)
    o = torch.zeros(B, S, H, hd, dtype=f, device=DEV)
    lse = torch.full((B, H, S), -math.inf, dtype=f, device=DEV)
    d = torch.zeros(B, S, H + 2 * Hkv, hd, dtype=f, device=DEV)
    ns = [S] * B if s["lengths"] is None else s["lengths"].tolist()
    for b in range(B):
        n = ns[b]
        if n == 0:
            continue
        k, v = (qkv[b, :n, a:a + Hkv].to(f).transpose(0, 1) for a in (H, H + Hkv))
        head = torch.arange(H, device=DEV) // (H // Hkv)
        step = max(64, min(n, (1 << 28) // (H * n)))
        for i0 in range(0, n, step):
            i1 = min(n, i0 + step)
            lo = max(0, i0 - c["window"] + 1)
            j = torch.cat([torch.arange(min(c["sinks"], lo), device=DEV), torch.arange(lo, i1, device=DEV)])
            i = torch.arange(i0, i1, device=DEV)[:, None]
            ok = (j <= i) & ((j > i - c["window"]) | (j < c["sinks"]))
            q = qkv[b, i0:i1, :H].to(f).transpose(0, 1)
            g = do[b, i0:i1].to(f).transpose(0, 1)
            kj, vj = k[head][:, j], v[head][:, j]
            x = (q @ kj.mT / math.sqrt(hd)).masked_fill(~ok, -math.inf)
            z = torch.logsumexp(x, -1)
            p = torch.exp(x - z[..., None])
            lse[b, :, i0:i1] = z / math.log(2.0)
            o[b, i0:i1] = (p @ vj).transpose(0, 1)
            dp = g @ vj.mT
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(hd)
            d[b, i0:i1, :H] = (ds @ kj).transpose(0, 1)
            for a, t in ((H, ds.mT @ q), (H + Hkv, p.mT @ g)):
                d[b, :, a:a + Hkv].index_add_(0, j, t.view(Hkv, H // Hkv, -1, hd).sum(1).transpose(0, 1))
    return {"o": o.view(B * S, -1), "lse": lse, "dqkv": d.view(B * S, -1)}


def _exact_step(c, s):
    """Sequence by sequence, from the list of positions that it sees."""
    f = torch.float64
    H, Hkv, hd, cap, sinks = c["H"], c["Hkv"], c["hd"], c["cap"], c["sinks"]
    turn = cap - sinks
    o = torch.zeros(c["B"], H, hd, dtype=f, device=DEV)
    cache = s["cache"].clone()
    for b, p in enumerate(s["pos"].tolist()):
        if p < 0:
            continue
        slot = lambda t: torch.where(t < sinks, t, sinks + (t - sinks) % turn)  # noqa: E731
        first = max(sinks, p - min(c["window"], turn) + 1)
        at = torch.cat([torch.arange(min(sinks, p + 1)), torch.arange(first, max(first, p + 1))]).to(DEV)
        cache[b, slot(torch.tensor(p)).item()] = s["qkv"][b, H * hd:]
        kv = cache[b, slot(at)].to(f).view(-1, 2, Hkv, hd)
        q = s["qkv"][b, :H * hd].to(f).view(Hkv, -1, hd)
        w = torch.softmax(q @ kv[:, 0].permute(1, 2, 0) / math.sqrt(hd), -1)
        o[b] = (w @ kv[:, 1].transpose(0, 1)).reshape(H, hd)
    return {"o": o.view(c["B"], -1), "cache": None}


def _exact_logprobs(c, s):
    f, V, T = torch.float64, c["V"], c["T"]
    out = {k: [] for k in ("logp", "entropy", "lse", "top_logp", "dlogits")}
    rows = max(1, (1 << 27) // V)
    for a in range(0, T, rows):
        x, t = s["logits"][a:a + rows, :V].to(f), s["targets"][a:a + rows]
        lp = torch.log_softmax(x, 1).masked_fill((x == -math.inf).all(1, keepdim=True), -math.inf)
        p = lp.exp()
        h = torch.special.entr(p).sum(1)
        one = torch.nn.functional.one_hot(t.clamp(min=0), V) if c["grad"] else None
        out["logp"].append(torch.where(t >= 0, lp[torch.arange(len(t), device=DEV), t.clamp(min=0)], 0.0))
        out["entropy"].append(h)
        out["lse"].append(torch.logsumexp(x, 1))
        if c["top"]:
            out["top_logp"].append(lp.topk(c["top"], 1).values)
        if c["grad"]:
            gl = (s["g_logp"][a:a + rows].to(f) * (t >= 0))[:, None]
            ge = s["g_entropy"][a:a + rows].to(f)[:, None]
            dh = torch.special.entr(p) - p * h[:, None]  # dH/dx = -p (log p + H)
            out["dlogits"].append((gl * (one - p) + ge * dh).float())
    out = {k: torch.cat(v) for k, v in out.items() if v}
    if c["top"]:
        out["top_ids"] = None
    return out


def _exact_dropout(c, s):
    import numpy as np

    n = c["rows"] * c["d"]
    m32, u = np.uint64(0xFFFFFFFF), np.uint64
    ctr = np.zeros((4, (n + 3) // 4), dtype=np.uint64)
    ctr[0] = np.arange(ctr.shape[1]) & 0xFFFFFFFF
    ctr[2], ctr[3] = s["stream"] % 2**32, s["stream"] // 2**32
    key = [s["seed"] % 2**32, s["seed"] // 2**32]
    for _ in range(10):
        a, b = u(0xD2511F53) * ctr[0], u(0xCD9E8D57) * ctr[2]
        ctr = np.stack([(b >> u(32)) ^ ctr[1] ^ u(key[0]), b & m32, (a >> u(32)) ^ ctr[3] ^ u(key[1]), a & m32])
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    kept = torch.from_numpy(ctr.T.reshape(-1)[:n] >= u(min(round(c["p"] * 2**32), 2**32 - 1)))
    kept = kept.view(c["rows"], c["d"]).to(DEV)
    y, dx = (s[k].double() * kept / (1.0 - c["p"]) for k in ("x", "dy"))
    return {"y": y if s["resid"] is None else y + s["resid"].double(), "dx": dx}


# ----------------------------------------------------------------------------- what a pass needs
def _pairs(c):
    """Visible (query, key) pairs of one sequence of the full length. A ragged
    batch is counted at its expected share: its lengths are drawn later."""
    S, W, K = c["S"], c["window"], c["sinks"]
    w = min(W, S)
    band = w * (w + 1) // 2 + (S - w) * w  # keys of the window
    out = max(0, S - W)  # queries with a key before their window; a sink is such a key
    first = min(K, out)
    return band + first * (first + 1) // 2 + max(0, out - K) * K


def work(case):
    c = case
    if c["op"] == "attention":
        rows, H, Hkv, hd = c["B"] * c["S"], c["H"], c["Hkv"], c["hd"]
        frac = 1.0 if c["lengths"] == "full" else 0.5
        qkv, o = rows * (H + 2 * Hkv) * hd * 2, rows * H * hd * 2
        # qkv and the output's gradient in; output, statistic and gradient out
        return {"bytes": frac * (2 * qkv + 2 * o + rows * H * 4),
                "flops": frac * 14 * c["B"] * H * hd * _pairs(c)}  # S, PV; dV, dP, dQ, dK and S again
    if c["op"] == "step":
        seen = min(c["window"], c["cap"] - c["sinks"]) + c["sinks"]
        n = c["longest"]
        mean = seen - seen * (seen - 1) / (2 * n) if n >= seen else (n + 1) / 2  # over drawn ages
        live = c["B"] - c["B"] // 7
        row = 2 * c["Hkv"] * c["hd"] * 2
        return {"bytes": live * (mean * row + row) + c["B"] * c["H"] * c["hd"] * 4,
                "flops": live * mean * 4 * c["H"] * c["hd"]}
    if c["op"] == "logprobs":
        n, e = c["T"] * c["V"], 2 if c["dtype"] == "bf16" else 4
        # the logits in once, and once more for a gradient that needs their sums first
        return {"bytes": n * e + (n * (e + 2) if c["grad"] else 0) + c["T"] * (24 + 12 * c["top"]),
                "flops": n * (4 + (6 if c["grad"] else 0))}
    n, e = c["rows"] * c["d"], 2 if c["dtype"] == "bf16" else 4
    return {"bytes": n * e * (4 + (1 if c["resid"] else 0)), "flops": 6 * n}
