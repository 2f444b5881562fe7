"""The operators over a KV cache in pages, as a serving program calls them.

"append" writes new tokens' K and V into the cache's pages, K (and Q) rotated to their positions on the way; "token"
is the attention of one new token per request over its pages; "verify" the tree-verification attention of packs whose
prefix lies in pages.

A pool is [n_pages, Hkv, page_size, D] (layout "hnd"), or a view of [n_pages, page_size, Hkv, D] ("nhd").  Lengths and
pack sizes follow from the case alone ("mix" seeds them), values, page order and trees from prepare()'s seed.  Slots
behind a request's last token hold NaN in the attention cases, as memory that nobody wrote may.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MAX_POS = 16384      # rows of the rotation table


def _append(B, s_lo, s_hi, n_lo, n_hi, ps, dtype="bf16", Hq=32, Hkv=8, D=128, rot=128, inter=False, pos=False,
            layout="hnd", mix=0):
    return dict(kind="append", B=B, s_lo=s_lo, s_hi=s_hi, n_lo=n_lo, n_hi=n_hi, ps=ps, dtype=dtype, Hq=Hq, Hkv=Hkv,
                D=D, rot=rot, inter=inter, pos=pos, layout=layout, mix=mix)


def _token(B, s_lo, s_hi, ps, dtype="bf16", Hq=32, Hkv=8, D=128, softcap=0.0, window=0, lse=False, layout="hnd",
           mix=0):
    return dict(kind="token", B=B, s_lo=s_lo, s_hi=s_hi, ps=ps, dtype=dtype, Hq=Hq, Hkv=Hkv, D=D, softcap=softcap,
                window=window, lse=lse, layout=layout, mix=mix)


def _verify(B, s_lo, s_hi, p_lo, p_hi, ps, dtype="bf16", Hq=32, Hkv=8, D=128, lse=False, layout="hnd", mix=0):
    return dict(kind="verify", B=B, s_lo=s_lo, s_hi=s_hi, p_lo=p_lo, p_hi=p_hi, ps=ps, dtype=dtype, Hq=Hq, Hkv=Hkv,
                D=D, lse=lse, layout=layout, mix=mix)


def listed():
    return [
        # the smallest call: one layer of one decode step of a batch, a token each
        dict(_append(8, 300, 2048, 1, 1, 64, mix=3), name="append-tokens-b8"),
        # prompts of a batch on their way into the cache, ragged
        dict(_append(6, 0, 0, 300, 4096, 64, mix=5), name="append-prompts-b6"),
        # an fp32 model that rotates part of the head in adjacent pairs, second half of a prompt, odd page size
        dict(_append(3, 1, 900, 37, 700, 24, dtype="fp32", Hq=16, Hkv=4, D=96, rot=32, inter=True, pos=True,
                     layout="nhd", mix=7), name="append-fp32-partial"),
        # one request of a chat, the latency of a decode step
        dict(_token(1, 2048, 2048, 64), name="token-b1-2k"),
        # an even batch at the benchmark's length
        dict(_token(8, 8192, 8192, 64), name="token-b8-8k"),
        # a server's batch, every length, small pages
        dict(_token(64, 300, 8192, 16, lse=True, layout="nhd", mix=11), name="token-ragged-b64"),
        # many short requests, head dim 64
        dict(_token(200, 1, 1024, 32, dtype="fp16", Hq=16, Hkv=4, D=64, mix=13), name="token-short-b200"),
        # one request over a long document: few heads, many keys
        dict(_token(1, 32768, 32768, 256), name="token-document-32k"),
        # head dim 256, scores capped by a tanh, layers that look back over a window
        dict(_token(8, 4096, 8192, 64, Hq=16, Hkv=8, D=256, softcap=50.0, window=4000, mix=17),
             name="token-d256-window"),
        # fp32 at a head dim that is no power of two, odd page size
        dict(_token(4, 500, 2000, 24, dtype="fp32", D=96, lse=True, mix=19), name="token-fp32-d96"),
        # verification of ragged packs over long prefixes
        dict(_verify(8, 1024, 8192, 32, 128, 64, lse=True, mix=3), name="verify-ragged-b8"),
        # a server's batch at the widths a cost-aware policy picks
        dict(_verify(32, 300, 4096, 2, 64, 128, dtype="fp16", layout="nhd", mix=5), name="verify-b32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [work(c) for c in listed()]
    while True:
        kind = rng.choices(["append", "token", "verify"], [3, 6, 2])[0]
        dtype = rng.choice(["bf16"] * 3 + ["fp16"] * 2 + ["fp32"])
        Hkv = rng.choice([8, 8, 8, 4, 2])
        Hq = Hkv * rng.choice([4, 4, 4, 8, 2, 1, 7])
        D = rng.choice([128] * 4 + [64] * 2 + [256, 96, 80])
        layout, mix = rng.choice(["hnd", "nhd"]), rng.randrange(1 << 20)
        ps = rng.choice([16, 32, 64, 64, 128, 256, rng.randint(1, 200)])
        heads = dict(dtype=dtype, Hq=Hq, Hkv=Hkv, D=D, layout=layout, mix=mix)
        if kind == "append":
            n_hi = rng.choice([1, _log_int(rng, 1, 4096)])
            n_lo = rng.randint(1, n_hi)
            s_hi = rng.choice([0, _log_int(rng, 1, 2048)])
            half = 4 if dtype == "fp32" else 8
            rot = rng.choice([0] + [r for r in range(2 * half, D + 1, 2 * half)][-4:])
            c = _append(_log_int(rng, 1, 64), rng.randint(0, s_hi), s_hi, n_lo, n_hi, ps, rot=rot,
                        inter=rng.random() < 0.3, pos=rng.random() < 0.3, **heads)
        elif kind == "token":
            s_hi = _log_int(rng, 1, 32768)
            s_lo = rng.choice([s_hi, rng.randint(1, s_hi)])
            c = _token(_log_int(rng, 1, 256), s_lo, s_hi, ps, softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                       window=rng.choice([0, 0, _log_int(rng, 1, 8192)]), lse=rng.random() < 0.3, **heads)
        else:
            s_hi = _log_int(rng, 1, 8192)
            s_lo = rng.choice([s_hi, rng.randint(1, s_hi)])
            p_hi = _log_int(rng, 1, 128)
            c = _verify(_log_int(rng, 1, 32), s_lo, s_hi, rng.randint(1, p_hi), p_hi,
                        64 * rng.choice([1, 1, 2, 3, 4]), lse=rng.random() < 0.3, **heads)
        w = work(c)
        pool = _pages(c).sum() * ps * Hkv * D * 2 * _esz(c) if kind == "append" else 0
        if w["flops"] <= max(x["flops"] for x in most) and w["bytes"] <= max(x["bytes"] for x in most) \
                and pool < 1 << 28:
            return c


# ---- sizes

def _esz(c):
    return 4 if c["dtype"] == "fp32" else 2


def _lengths(c):
    """Cached tokens S and new tokens N of every request."""
    rng = np.random.default_rng(c["mix"])
    S = rng.integers(c["s_lo"], c["s_hi"] + 1, size=c["B"])
    lo, hi = (c["n_lo"], c["n_hi"]) if c["kind"] == "append" else \
        (c["p_lo"], c["p_hi"]) if c["kind"] == "verify" else (0, 0)
    return S.astype(np.int64), rng.integers(lo, hi + 1, size=c["B"]).astype(np.int64)


def _pages(c):
    S, N = _lengths(c)
    return -(-(S + (N if c["kind"] == "append" else 0)) // c["ps"])


def _seen(c, S):
    """First visible key of every request's new token."""
    return np.maximum(S - c["window"], 0) if c["window"] else np.zeros_like(S)


def work(c):
    S, N = _lengths(c)
    e, D, Hq, Hkv = _esz(c), c["D"], c["Hq"], c["Hkv"]
    ids = int(_pages(c).sum()) * 4
    if c["kind"] == "append":
        T = int(N.sum())
        return {"bytes": T * ((4 * Hkv + 2 * Hq) * D * e + c["rot"] * 4) + 8 * c["B"],
                "flops": T * (Hq + Hkv) * c["rot"] * 3}
    if c["kind"] == "token":
        n = int((S - _seen(c, S)).sum())
        return {"bytes": n * Hkv * D * 2 * e + c["B"] * Hq * (2 * D * e + (4 if c["lse"] else 0)) + ids,
                "flops": 4 * n * Hq * D}
    T = int(N.sum())
    return {"bytes": int((S + N).sum()) * Hkv * D * 2 * e + T * (Hq * (2 * D * e + (4 if c["lse"] else 0)) + 16) + ids,
            "flops": int((4 * N * (S + N)).sum()) * Hq * D}


# ---- inputs

def _tree_words(rng, P):
    """Ancestor words [sum P, 2] of random trees whose nodes favour early parents, as a best-first search's do."""
    rows = []
    for n in P:
        words = []
        for i in range(int(n)):
            up = words[int(i * rng.random() ** 1.5)] if i else 0
            words.append(up | 1 << i)
        rows += [(w & (1 << 64) - 1, w >> 64) for w in words]
    return torch.from_numpy(np.array(rows, dtype=np.uint64).view(np.int64))


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    S, N = _lengths(c)
    dt, D, Hq, Hkv, ps, B = DTYPES[c["dtype"]], c["D"], c["Hq"], c["Hkv"], c["ps"], c["B"]

    def normal(*shape, scale=None):
        x = torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)
        return (x if scale is None else x * scale).to(dt)

    # channels of K differ in size, a few stand out; Q is such that scores spread over a few units
    chan = torch.exp(0.4 * torch.randn(Hkv, 1, D, generator=g, device=DEV))
    chan[:, :, :: max(D // 2, 1)] *= 4.0
    q_scale = 2.0 / float(chan.square().mean().sqrt())

    need = _pages(c)
    n_pages = int(need.sum()) + 3
    order = rng.permutation(n_pages)
    width = max(int(need.max()), 1) + 1
    table = np.full((B, width), -1, dtype=np.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += int(need[b])
    table_dev = torch.from_numpy(table).to(DEV)

    def pool(scale):
        if c["layout"] == "hnd":
            return normal(n_pages, Hkv, ps, D, scale=scale)
        return normal(n_pages, ps, Hkv, D, scale=None if scale is None else scale[:, 0]).transpose(1, 2)

    st = dict(case=c, S=S, N=N, kp=pool(chan), vp=pool(None), table=table_dev,
              seq_len=torch.from_numpy(S.astype(np.int32)).to(DEV))
    cu = np.concatenate([[0], np.cumsum(N)]).astype(np.int32)
    T = int(cu[-1])
    if c["kind"] == "append":
        st.update(q=normal(T, Hq, D, scale=q_scale), k=normal(T, Hkv, D, scale=chan[:, 0]), v=normal(T, Hkv, D),
                  cu_q=None if N.max() == 1 else torch.from_numpy(cu).to(DEV), cos=None, sin=None, positions=None)
        slots = np.concatenate([s + np.arange(n) for s, n in zip(S, N)])
        owner = np.repeat(np.arange(B), N)
        st["page"] = torch.from_numpy(table[owner, slots // ps].astype(np.int64)).to(DEV)
        st["offset"] = torch.from_numpy((slots % ps).astype(np.int64)).to(DEV)
        where = slots
        if c["rot"] and c["pos"]:
            # positions of their own, as a pack's depths or a shifted context have them
            where = np.minimum(slots + rng.integers(0, 4096, size=T), MAX_POS - 1)
            st["positions"] = torch.from_numpy(where.astype(np.int32)).to(DEV)
        st["where"] = torch.from_numpy(where.astype(np.int64)).to(DEV)
        if c["rot"]:
            angle = torch.arange(MAX_POS, dtype=torch.float64)[:, None] \
                * 10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64) / c["rot"])
            st["cos"], st["sin"] = angle.cos().float().to(DEV), angle.sin().float().to(DEV)
        return st
    # what lies behind a request's last token was never written
    for b in range(B):
        if S[b] % ps:
            for x in (st["kp"], st["vp"]):
                x[int(table[b, need[b] - 1]), :, int(S[b] % ps):] = float("nan")
    if c["kind"] == "token":
        st["q"] = normal(B, Hq, D, scale=q_scale)
        return st
    st.update(q=normal(T, Hq, D, scale=q_scale), k=normal(Hkv, T, D, scale=chan), v=normal(Hkv, T, D), cu=cu,
              cu_q=torch.from_numpy(cu).to(DEV), pack_len=torch.from_numpy(N.astype(np.int32)).to(DEV),
              words=_tree_words(rng, N).to(DEV), total_kv=int((S + N).sum()))
    return st


# ---- one pass

def run(st):
    c = st["case"]
    return {"append": _run_append, "token": _run_token, "verify": _run_verify}[c["kind"]](st, c)


def _rotate(x, cos, sin, c):
    """x [T, H, D] with the first rot elements of each head turned by the token's angles."""
    rot = c["rot"]
    x = x.float()
    cos, sin = cos[:, None], sin[:, None]
    if c["inter"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _run_append(st, c):
    if own:
        from cast_amd import paged_append
        q, new_len = paged_append(st["k"], st["v"], st["kp"], st["vp"], st["table"], st["seq_len"], st["cu_q"],
                                  q=st["q"], cos=st["cos"], sin=st["sin"], positions=st["positions"],
                                  interleaved=c["inter"])
        return dict(q=q, new_len=new_len, k_pages=st["kp"], v_pages=st["vp"])
    q, k, dt = st["q"], st["k"], st["k"].dtype
    if c["rot"]:
        cos, sin = st["cos"][st["where"]], st["sin"][st["where"]]
        q, k = _rotate(q, cos, sin, c).to(dt), _rotate(k, cos, sin, c).to(dt)
    st["kp"][st["page"], :, st["offset"]] = k
    st["vp"][st["page"], :, st["offset"]] = st["v"]
    n = 1 if st["cu_q"] is None else st["cu_q"][1:] - st["cu_q"][:-1]
    return dict(q=q, new_len=st["seq_len"] + n, k_pages=st["kp"], v_pages=st["vp"])


def _pages_of(st, x, b, lo, hi):
    """Keys [lo, hi) of request b: [Hkv, hi - lo, D] in 32 bits."""
    ps = st["case"]["ps"]
    first, last = lo // ps, -(-hi // ps)
    y = x[st["table"][b, first:last].long()].transpose(0, 1).flatten(1, 2)
    return y[:, lo - first * ps:hi - first * ps].float()


def _softmax_values(s, v):
    """Weights of scores s over the last axis, applied to v, and the log of their sum."""
    m = s.max(dim=-1, keepdim=True).values
    p = (s - m).exp()
    l = p.sum(dim=-1, keepdim=True)
    return torch.matmul(p, v) / l, (m + l.log())[..., 0]


def _run_token(st, c):
    if own:
        from cast_amd import paged_attention
        return paged_attention(st["q"], st["kp"], st["vp"], st["table"], st["seq_len"], softcap=c["softcap"],
                               window=c["window"], return_lse=c["lse"])
    Hkv, D, q = c["Hkv"], c["D"], st["q"]
    out, lse = [], []
    for b, (lo, n) in enumerate(zip(_seen(c, st["S"]).tolist(), st["S"].tolist())):
        k, v = _pages_of(st, st["kp"], b, lo, n), _pages_of(st, st["vp"], b, lo, n)
        s = torch.matmul(q[b].view(Hkv, -1, D).float(), k.transpose(1, 2).contiguous()) / math.sqrt(D)
        if c["softcap"]:
            s = c["softcap"] * torch.tanh(s / c["softcap"])
        o, l = _softmax_values(s, v)
        out.append(o.flatten(0, 1))
        lse.append(l.flatten())
    out = torch.stack(out).to(q.dtype)
    return (out, torch.stack(lse)) if c["lse"] else out


def _run_verify(st, c):
    if own:
        from cast_amd import paged_tree_attention
        return paged_tree_attention(st["q"], st["kp"], st["vp"], st["table"], st["k"], st["v"], st["cu_q"],
                                    st["seq_len"], st["pack_len"], st["words"], total_kv=st["total_kv"],
                                    return_lse=c["lse"])
    Hkv, D, q = c["Hkv"], c["D"], st["q"]
    out, lse = [], []
    for b, (n, p) in enumerate(zip(st["S"].tolist(), st["N"].tolist())):
        a, e = int(st["cu"][b]), int(st["cu"][b + 1])
        k = torch.cat([_pages_of(st, st["kp"], b, 0, n), st["k"][:, a:e].float()], dim=1)
        v = torch.cat([_pages_of(st, st["vp"], b, 0, n), st["v"][:, a:e].float()], dim=1)
        qb = q[a:e].transpose(0, 1).reshape(Hkv, -1, D).float()          # rows (query head of the group, token)
        s = torch.matmul(qb, k.transpose(1, 2).contiguous()).view(Hkv, -1, p, n + p) / math.sqrt(D)
        j = torch.arange(p, device=DEV)
        bits = st["words"][a:e][:, j // 64] >> (j % 64) & 1
        s[..., n:].masked_fill_(bits == 0, float("-inf"))
        o, l = _softmax_values(s.flatten(1, 2), v)
        out.append(o.view(-1, p, D).transpose(0, 1))
        lse.append(l.view(-1, p).transpose(0, 1))
    out = torch.cat(out).to(q.dtype)
    return (out, torch.cat(lse)) if c["lse"] else out


# ---- the definition, in 64 bits

def _turn(x, angle_cos, angle_sin, c):
    """Rotation by complex products: element pairs as (real, imaginary)."""
    rot = c["rot"]
    y = x.double().clone()
    i = torch.arange(rot // 2, device=DEV)
    re, im = (2 * i, 2 * i + 1) if c["inter"] else (i, i + rot // 2)
    z = torch.complex(y[..., re], y[..., im]) * torch.complex(angle_cos, angle_sin)[:, None]
    y[..., re], y[..., im] = z.real, z.imag
    return y


def exact(c, seed):
    st = prepare(c, seed)
    S, N, ps, Hkv, G, D = st["S"], st["N"], c["ps"], c["Hkv"], c["Hq"] // c["Hkv"], c["D"]
    if c["kind"] == "append":
        q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
        if c["rot"]:
            cs = [st[x].double()[st["where"]] for x in ("cos", "sin")]
            q, k = _turn(q, *cs, c), _turn(k, *cs, c)
        kp, vp = st["kp"].double(), st["vp"].double()
        for pool, x in ((kp, k), (vp, v)):
            rows = pool.transpose(1, 2).reshape(-1, Hkv, D)              # a copy, one row per slot of the cache
            rows[st["page"] * ps + st["offset"]] = x
            pool.copy_(rows.view(-1, ps, Hkv, D).transpose(1, 2))
        return dict(q=q, new_len=torch.from_numpy((S + N).astype(np.int32)).to(DEV), k_pages=kp, v_pages=vp)

    def slots(x, b, lo, hi):
        t = torch.arange(lo, hi, device=DEV)
        return x[st["table"][b].long()[t // ps], :, t % ps].double().transpose(0, 1).contiguous()   # [Hkv, n, D]

    def attend(q, k, v, hidden=None):
        """q [rows, Hq, D] against k, v [Hkv, n, D]; hidden [rows, n]."""
        out, lse = [], []
        for h in range(c["Hq"]):
            s = k[h // G] @ q[:, h].double().t().contiguous() * D ** -0.5                          # [n, rows]
            if c.get("softcap"):
                s = torch.tanh(s / c["softcap"]) * c["softcap"]
            if hidden is not None:
                s = s.masked_fill(hidden.t(), float("-inf"))
            l = torch.logsumexp(s, dim=0)
            out.append(torch.exp(s - l).t().contiguous() @ v[h // G])
            lse.append(l)
        return torch.stack(out, 1), torch.stack(lse, 1)

    got = []
    for b in range(c["B"]):
        if c["kind"] == "token":
            lo = max(int(S[b]) - c["window"], 0) if c["window"] else 0
            got.append(attend(st["q"][b:b + 1], slots(st["kp"], b, lo, int(S[b])), slots(st["vp"], b, lo, int(S[b]))))
            continue
        a, e = int(st["cu"][b]), int(st["cu"][b + 1])
        k, v = (torch.cat([slots(x, b, 0, int(S[b])), y[:, a:e].double()], dim=1)
                for x, y in ((st["kp"], st["k"]), (st["vp"], st["v"])))
        hidden = torch.zeros(e - a, int(S[b]) + e - a, dtype=torch.bool)
        for i, (w0, w1) in enumerate(st["words"][a:e].cpu().numpy().view(np.uint64).tolist()):
            w = w0 | w1 << 64
            hidden[i, int(S[b]):] = torch.tensor([not w >> j & 1 for j in range(e - a)])
        got.append(attend(st["q"][a:e], k, v, hidden.to(DEV)))
    out, lse = torch.cat([o for o, _ in got]), torch.cat([l for _, l in got])
    return (out, lse) if c["lse"] else out
