"""The paged KV cache on the GPU: append with rotation and one-token attention
against the 64-bit restatement in oracle/paged.py.

Bounds, with u = 2^-23 (float, either rounding direction):
  scores     a sum of D exact or once-rounded products: (D + 4) u * terms, the
             scaling and a tanh's cap twice more of the score, itself at most terms
  weights    2 * (score error) + (n + 64) u for the sums and the exponential;
             16-bit weights are two terms, at most 2^-16 of the weight off
  output     that share of sum(weight * |v|), plus half a step of the type
  lse        score error + (n + 64) u + 2 u |lse|
"""
import numpy as np
import pytest
import torch

from oracle import paged as OP

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def make_cache(gpu, lens, Hkv, D, ps, dtype, layout="hnd", seed=0, spare=2, garbage=float("nan"), chan=1.0):
    """Pools with shuffled pages, garbage in every slot behind a request's last, and their table."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // ps) for n in lens]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g).tolist()
    width = max(max(need), 1) + 1
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    shape = (n_pages, Hkv, ps, D) if layout == "hnd" else (n_pages, ps, Hkv, D)
    pools = []
    for scale in (chan, 1.0):
        x = (torch.randn(shape, generator=g) * scale).to(DT[dtype])
        pools.append(x if layout == "hnd" else x.transpose(1, 2))
    at = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = torch.tensor(order[at:at + need[b]], dtype=torch.int32)
        at += need[b]
        if n > 0 and n % ps:
            for x in pools:
                x[int(table[b, need[b] - 1]), :, n % ps:] = garbage
    for i in order[at:]:
        for x in pools:
            x[i] = garbage
    return (*pools, table, g)


def check_attention(got, lse, ref, dtype, n, D):
    out, rl, spread, terms = ref
    # terms is per (request, head): the score bound of its keys
    score = ((D + 4) * U + 4 * U) * terms
    w = 2 * score + (n + 64) * U + (2.0 ** -16 if dtype != torch.float32 else 0.0)
    bound = w[..., None] * spread + HALF[dtype] * out.abs() + 2.0 ** -24 * (dtype == torch.float16)
    err = (got.double().cpu() - out).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"out off by {(err / bound.clamp_min(1e-300)).max():.2f} bounds"
    if lse is not None:
        lb = score + (n + 64) * U + 2 * U * rl.abs()
        ok = (lse.double().cpu() - rl).abs() <= lb
        assert (ok | (torch.isneginf(rl) & torch.isneginf(lse.cpu()))).all()


CASES = [
    # dtype, Hq, Hkv, D, page size, layout, lengths, window, softcap, kv_split
    ("bf16", 8, 2, 128, 64, "hnd", [1, 2, 63, 64, 65, 300], 0, 0.0, 0),
    ("bf16", 8, 2, 128, 16, "nhd", [1, 15, 16, 17, 129, 1000], 0, 0.0, 128),
    ("fp16", 8, 2, 128, 32, "hnd", [128, 127, 511, 700], 0, 30.0, 256),
    ("fp32", 8, 2, 128, 64, "nhd", [1, 63, 64, 65, 333], 0, 5.0, 64),
    ("bf16", 4, 4, 64, 48, "hnd", [1, 47, 48, 49, 500], 0, 0.0, 0),
    ("fp16", 7, 1, 64, 16, "nhd", [5, 900], 0, 0.0, 0),
    ("fp32", 6, 2, 64, 1, "hnd", [1, 2, 100, 260], 0, 0.0, 0),
    ("bf16", 4, 2, 256, 64, "hnd", [1, 130, 400], 0, 0.0, 128),
    ("fp16", 2, 2, 256, 16, "nhd", [33, 257], 100, 20.0, 0),
    ("fp32", 4, 1, 256, 32, "hnd", [31, 200], 0, 0.0, 64),
    ("bf16", 4, 2, 96, 24, "nhd", [1, 23, 24, 25, 400], 0, 0.0, 128),
    ("fp16", 4, 2, 80, 7, "hnd", [6, 7, 8, 222], 50, 0.0, 0),
    ("fp32", 4, 2, 96, 24, "hnd", [25, 301], 130, 10.0, 64),
    ("bf16", 4, 2, 8, 16, "hnd", [40], 0, 0.0, 0),
    ("fp32", 4, 2, 40, 16, "nhd", [140], 0, 0.0, 0),
    ("bf16", 4, 2, 200, 33, "hnd", [150, 3], 0, 0.0, 0),
    ("bf16", 40, 2, 128, 64, "hnd", [300, 17], 0, 0.0, 128),      # 20 query heads a KV head: two blocks of 16
    ("fp32", 33, 1, 64, 20, "hnd", [130], 0, 0.0, 64),
    ("bf16", 8, 2, 128, 64, "hnd", [700, 10, 129], 1, 0.0, 128),   # windows of one, inside and across tiles
    ("fp16", 8, 2, 128, 16, "hnd", [700, 300, 129, 128], 130, 0.0, 128),
    ("bf16", 8, 2, 128, 200, "nhd", [399, 400, 401, 199], 0, 50.0, -1),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:6]) + f"-w{c[7]}-c{c[8]}-s{c[9]}")
def test_attention_matches_64_bits(gpu, case):
    from cast_amd import paged_attention
    dtype, Hq, Hkv, D, ps, layout, lens, window, softcap, split = case
    print("case attention", case, flush=True)
    kp, vp, table, g = make_cache(gpu, lens, Hkv, D, ps, dtype, layout, seed=len(lens) + D)
    q = (torch.randn((len(lens), Hq, D), generator=g) * 2).to(DT[dtype])
    ref = OP.attention(q, kp, vp, table, lens, softcap=softcap, window=window)
    dev = lambda x: x.to(gpu)
    kd = dev(kp) if layout == "hnd" else dev(kp.transpose(1, 2).contiguous()).transpose(1, 2)
    vd = dev(vp) if layout == "hnd" else dev(vp.transpose(1, 2).contiguous()).transpose(1, 2)
    out, lse = paged_attention(dev(q), kd, vd, dev(table), torch.tensor(lens, dtype=torch.int32, device=gpu),
                               softcap=softcap, window=window, kv_split=split, return_lse=True, check=True)
    check_attention(out, lse, ref, DT[dtype], max(lens), D)


def test_large_batch_of_short_and_empty_requests(gpu):
    # more requests than one wave looks at, lengths of zero among them
    from cast_amd import paged_attention
    rng = np.random.default_rng(3)
    lens = [int(x) for x in rng.integers(0, 40, size=150)]
    lens[0] = lens[64] = lens[149] = 0
    lens[70] = 900
    kp, vp, table, g = make_cache(gpu, lens, 2, 64, 16, "bf16", seed=5)
    q = torch.randn((150, 4, 64), generator=g).to(torch.bfloat16)
    ref = OP.attention(q, kp, vp, table, lens)
    out, lse = paged_attention(q.to(gpu), kp.to(gpu), vp.to(gpu), table.to(gpu), lens, return_lse=True, check=True)
    check_attention(out, lse, ref, torch.bfloat16, 900, 64)
    empty = torch.tensor([n == 0 for n in lens])
    assert (out.cpu()[empty] == 0).all() and torch.isneginf(lse.cpu()[empty]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("ps", [16, 24])
def test_bad_requests_give_zeros_and_leave_the_others(gpu, dtype, ps):
    from cast_amd import paged_attention
    lens = [300, 300, 300, 300, 300]
    kp, vp, table, g = make_cache(gpu, lens, 2, 64, ps, dtype, seed=1)
    q = torch.randn((5, 4, 64), generator=g).to(DT[dtype])
    ref = OP.attention(q, kp, vp, table, lens)
    table = table.clone()
    table[1, 3] = -1                          # in the middle: one split sees it
    table[2, 0] = kp.shape[0]                 # just past the pool
    said = [300, 300, 300, table.shape[1] * ps + 1, -5]
    for split in (64, -1, 0):
        args = (q.to(gpu), kp.to(gpu), vp.to(gpu), table.to(gpu), torch.tensor(said, dtype=torch.int32, device=gpu))
        out, lse = paged_attention(*args, kv_split=split, return_lse=True)
        keep = tuple(x[:1] for x in ref)
        check_attention(out[:1], lse[:1], keep, DT[dtype], 300, 64)
        assert (out[1:] == 0).all() and torch.isneginf(lse[1:]).all()
        with pytest.raises(ValueError, match="page id.*|.*page id"):
            paged_attention(*args, kv_split=split, check=True)
    # pages in front of a window may be gone
    free = table.clone()
    free[:, :2] = -1
    win = 300 - 2 * ps
    ref = OP.attention(q[:1], kp, vp, table[:1], [300], window=win)
    out, lse = paged_attention(q[:1].to(gpu), kp.to(gpu), vp.to(gpu), free[:1].to(gpu), [300], window=win,
                               return_lse=True, check=True)
    check_attention(out, lse, ref, DT[dtype], 300, 64)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_infinities_and_nan_reach_only_who_sees_them(gpu, dtype):
    from cast_amd import paged_attention
    lens = [130, 130, 130, 130]
    kp, vp, table, g = make_cache(gpu, lens, 2, 64, 16, dtype, seed=2)
    q = torch.randn((4, 4, 64), generator=g).to(DT[dtype])
    clean = OP.attention(q, kp, vp, table, lens)
    vp[int(table[1, 2]), 0, 3, 5] = float("inf")       # one element of KV head 0 of request 1
    kp[int(table[2, 8]), 1, 1, 0] = float("nan")       # KV head 1 of request 2, the last visible key
    kp[int(table[3, 0]), 0, 0, :] = 0
    kp[int(table[3, 0]), 0, 0, 0] = float("inf")       # scores of +-inf in KV head 0 of request 3
    out, lse = paged_attention(q.to(gpu), kp.to(gpu), vp.to(gpu), table.to(gpu), lens, return_lse=True, kv_split=128)
    o, l = out.cpu(), lse.cpu()
    sane = torch.ones((4, 4, 64), dtype=torch.bool)
    sane[1, :2, 5] = sane[2, 2:] = sane[3, :2] = False
    keep = [clean[0].clone(), clean[2]]
    got = torch.where(sane, o.double(), keep[0])
    check_attention(got.to(DT[dtype]), None, (keep[0], clean[1], clean[2], clean[3]), DT[dtype], 130, 64)
    assert torch.isinf(o[1, :2, 5]).all() and torch.isnan(o[2, 2:]).all() and torch.isnan(l[2, 2:]).all()
    for h in range(2):
        if q[3, h, 0] > 0:
            assert torch.isnan(o[3, h]).all()          # a score of +inf
        elif q[3, h, 0] < 0:
            assert torch.isfinite(o[3, h]).all()       # -inf: that key weighs nothing


def test_a_row_of_lowest_scores_has_no_weight(gpu):
    # every visible score is -inf: zeros and lse = -inf, as for no visible key
    from cast_amd import paged_attention
    kp = torch.full((2, 1, 16, 64), float("-inf"), dtype=torch.bfloat16, device=gpu)
    vp = torch.ones_like(kp)
    q = torch.full((1, 1, 64), 1.0, dtype=torch.bfloat16, device=gpu)
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=gpu)
    out, lse = paged_attention(q, kp, vp, table, [20], return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    # the type's lowest value in one element: finite scores far apart
    kp.fill_(0)
    kp[0, 0, 3, 0] = torch.finfo(torch.bfloat16).min
    out, lse = paged_attention(q, kp, vp, table, [20], return_lse=True)
    assert (out == 1).all() and abs(lse.item() - np.log(19)) < 1e-5


def test_the_store_is_a_pool_of_one_page_per_request(gpu):
    # [B, Hkv, cap, D] with a capacity that is no multiple of anything
    from cast_amd import paged_attention
    cap, lens = 203, [203, 1, 150]
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn((3, 2, cap, 128), generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((3, 8, 128), generator=g).to(torch.bfloat16)
    table = torch.arange(3, dtype=torch.int32)[:, None]
    ref = OP.attention(q, k, v, table, lens)
    for split in (0, 128):
        out, lse = paged_attention(q.to(gpu), k.to(gpu), v.to(gpu), table.to(gpu), lens, return_lse=True, check=True,
                                   kv_split=split)
        check_attention(out, lse, ref, torch.bfloat16, cap, 128)


def test_strided_and_unaligned_inputs(gpu):
    # q out of a fused projection, an output inside a larger tensor, a table that is a slice of a wider one
    from cast_amd import paged_attention
    lens = [70, 200]
    kp, vp, table, g = make_cache(gpu, lens, 2, 128, 16, "bf16", seed=6)
    qkv = torch.randn((2, 3, 8, 128), generator=g).to(torch.bfloat16)
    wide = torch.full((2, table.shape[1] + 5), 99999, dtype=torch.int32)
    wide[:, 2:2 + table.shape[1]] = table
    ref = OP.attention(qkv[:, 1], kp, vp, table, lens)
    big = torch.full((2, 16, 128), 7.0, dtype=torch.bfloat16, device=gpu)
    out, lse = paged_attention(qkv.to(gpu)[:, 1], kp.to(gpu), vp.to(gpu), wide.to(gpu)[:, 2:2 + table.shape[1]], lens,
                               out=big[:, 4:12], return_lse=True, check=True)
    check_attention(big[:, 4:12], lse, ref, torch.bfloat16, 200, 128)
    assert (big[:, :4] == 7).all() and (big[:, 12:] == 7).all()
    odd = torch.randn(2 * 8 * 128 + 1, generator=g).to(torch.bfloat16).to(gpu)[1:].view(2, 8, 128)
    a = paged_attention(odd, kp.to(gpu), vp.to(gpu), table.to(gpu), lens)
    b = paged_attention(odd.clone(), kp.to(gpu), vp.to(gpu), table.to(gpu), lens)
    assert torch.equal(a, b)


def test_offsets_past_32_bits(gpu):
    # one page of 1.3 M slots (2.6 GB of K and of V) and a pool whose last pages lie past 4 GB
    from cast_amd import paged_append, paged_attention
    cap = 1300003
    k = torch.zeros((1, cap, 8, 128), dtype=torch.bfloat16, device=gpu).transpose(1, 2)
    v = torch.zeros_like(k.transpose(1, 2)).transpose(1, 2)
    g = torch.Generator().manual_seed(8)
    rows = torch.randn((2, 40, 8, 128), generator=g).to(torch.bfloat16).to(gpu)
    n0 = cap - 40
    table = torch.zeros((1, 1), dtype=torch.int32, device=gpu)
    _, new_len = paged_append(rows[0], rows[1], k, v, table, [n0], [0, 40], check=True)
    assert new_len.tolist() == [cap]
    assert torch.equal(k[0, :, n0:].transpose(0, 1), rows[0]) and torch.equal(v[0, :, n0:].transpose(0, 1), rows[1])
    q = torch.randn((1, 8, 128), generator=g).to(torch.bfloat16)
    out, lse = paged_attention(q.to(gpu), k, v, table, new_len, window=40, return_lse=True, check=True)
    pool = rows.cpu().transpose(1, 2).contiguous()
    ref = OP.attention(q, pool[:1], pool[1:], torch.zeros((1, 1), dtype=torch.int32), [40])
    check_attention(out, lse, ref, torch.bfloat16, 40, 128)
    del k, v
    big = torch.empty((5000, 8, 64, 1024), dtype=torch.bfloat16, device=gpu)   # 5 GB
    kp, vp = big[:, :4, :, :128], big[:, 4:, :, 512:640]
    ids = torch.tensor([[4999, 4998]], dtype=torch.int32)
    rows = torch.randn((2, 100, 4, 128), generator=g).to(torch.bfloat16)
    _, new_len = paged_append(rows[0].to(gpu), rows[1].to(gpu), kp, vp, ids.to(gpu), [0], [0, 100], check=True)
    q = torch.randn((1, 4, 128), generator=g).to(torch.bfloat16)
    out, lse = paged_attention(q.to(gpu), kp, vp, ids.to(gpu), new_len, return_lse=True, check=True)
    pool = rows.transpose(1, 2).contiguous()
    ref = OP.attention(q, pool[:1], pool[1:], torch.zeros((1, 1), dtype=torch.int32), [100])
    check_attention(out, lse, ref, torch.bfloat16, 100, 128)


# ---- append

def tables(max_pos, rot, gpu):
    angle = torch.arange(max_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2).double() / rot)
    return angle.cos().float(), angle.sin().float()


def check_rows(got, ref, size, dtype):
    """got (the type) against 64-bit rows; size: the sum of the two products' sizes."""
    bound = HALF[dtype] * ref.abs() + 2 * U * size + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    err = (got.double().cpu() - ref).abs()
    assert (err <= bound).all(), f"{(err / bound.clamp_min(1e-300)).max():.2f} bounds"


APPENDS = [
    # dtype, Hq, Hkv, D, page size, layout, seq_len, new rows, rot, interleaved, explicit positions
    ("bf16", 8, 2, 128, 64, "hnd", [0, 63, 64, 130], [1, 1, 1, 1], 128, False, False),
    ("bf16", 8, 2, 128, 16, "nhd", [0, 5, 16, 17], [40, 0, 1, 33], 128, False, False),
    ("fp16", 4, 4, 64, 7, "hnd", [3, 0], [20, 15], 64, True, True),
    ("fp32", 4, 2, 96, 24, "nhd", [23, 0, 1], [2, 50, 0], 32, True, True),
    ("fp32", 4, 2, 40, 16, "hnd", [0, 9], [17, 30], 24, False, False),
    ("bf16", 14, 2, 80, 1, "hnd", [2, 0], [5, 6], 48, False, True),
    ("fp16", 2, 1, 256, 32, "nhd", [31], [70], 0, False, False),
    ("bf16", 40, 8, 128, 128, "hnd", [100], [60], 64, False, False),
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "-".join(str(x) for x in c[:6]) + f"-r{c[8]}-{c[9]}-{c[10]}")
def test_append_matches_64_bits(gpu, case):
    from cast_amd import paged_append
    dtype, Hq, Hkv, D, ps, layout, seq, new, rot, inter, pos = case
    print("case append", case, flush=True)
    dt = DT[dtype]
    B, total, tail = len(seq), sum(new), 3
    kp, vp, table, g = make_cache(gpu, [s + n for s, n in zip(seq, new)], Hkv, D, ps, dtype, layout, seed=D, garbage=1.5)
    q, k, v = (torch.randn((total + tail, h, D), generator=g).to(dt) for h in (Hq, Hkv, Hkv))
    cu = [0] + list(np.cumsum(new))
    slots = [s + j for s, n in zip(seq, new) for j in range(n)]
    cos = sin = positions = None
    if rot:
        cos, sin = tables(400, rot, gpu)
        if pos:
            positions = torch.randint(0, 400, (total + tail,), generator=g, dtype=torch.int32)
            slots = positions[:total].tolist()
    one = all(n == 1 for n in new)
    if one:
        q, k, v = q[:total], k[:total], v[:total]
        tail = 0
    if rot:
        cq, sq = cos[slots], sin[slots]
        qr, qsize = OP.rotate(q[:total], cq, sq, inter)
        kr, ksize = OP.rotate(k[:total], cq, sq, inter)
    else:
        qr, kr = q[:total].double(), k[:total].double()
        qsize, ksize = torch.zeros_like(qr), torch.zeros_like(kr)
    want_k, want_v = OP.append(kp, kr, table, seq, cu), OP.append(vp, v, table, seq, cu)
    size_k = OP.append(torch.zeros_like(kp), ksize, table, seq, cu)
    dev = lambda x: None if x is None else x.to(gpu)
    kd, vd = (dev(x.transpose(1, 2).contiguous()).transpose(1, 2) if layout == "nhd" else dev(x) for x in (kp, vp))
    q_out = torch.full((total + tail, Hq, D), 9.0, dtype=dt, device=gpu)
    k_out = torch.full((total + tail, Hkv, D), 9.0, dtype=dt, device=gpu)
    got_q, new_len = paged_append(dev(k), dev(v), kd, vd, dev(table), torch.tensor(seq, dtype=torch.int32, device=gpu),
                                  None if one else torch.tensor(cu, dtype=torch.int32, device=gpu), q=dev(q),
                                  cos=dev(cos), sin=dev(sin), positions=dev(positions), interleaved=inter, q_out=q_out,
                                  k_out=k_out, check=True)
    assert got_q is q_out and new_len.tolist() == [s + n for s, n in zip(seq, new)]
    check_rows(q_out[:total], qr, qsize, dt)
    check_rows(k_out[:total], kr, ksize, dt)
    assert (q_out[total:] == 9).all() and (k_out[total:] == 9).all()     # rows behind the last request
    check_rows(kd, want_k, size_k, dt)
    assert torch.equal(vd.double().cpu(), want_v)
    # in place, on strided inputs: the same bits
    qi, ki = (torch.cat([x, x], dim=-1).to(gpu)[..., :D] for x in (q, k))
    paged_append(ki, dev(v), kd, vd, dev(table), seq, None if one else cu, q=qi, cos=dev(cos), sin=dev(sin),
                 positions=dev(positions), interleaved=inter, q_out=qi, k_out=ki)
    assert torch.equal(qi[:total], q_out[:total]) and torch.equal(ki[:total], k_out[:total])


def test_rejected_rows_leave_everything_as_it_was(gpu):
    from cast_amd import paged_append
    ps, D = 16, 64
    table = torch.tensor([[0, 1, 2], [3, -1, 4], [5, 99, 6], [7, 8, 9], [10, 11, 12]], dtype=torch.int32)
    seq = [30, 14, 14, 47, -2]
    new = [5, 5, 5, 2, 1]                     # request 3 passes its table, 1 and 2 meet a bad page, 4 has no length
    cu = [0, 5, 10, 15, 17, 18]
    g = torch.Generator().manual_seed(0)
    k, v, q = (torch.randn((18, 2, D), generator=g).to(torch.bfloat16).to(gpu) for _ in range(3))
    kp, vp = (torch.full((13, 2, ps, D), 3.0, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    qo, ko = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
    args = (k, v, kp, vp, table.to(gpu), seq, cu)
    _, new_len = paged_append(*args, q=q, q_out=qo, k_out=ko)
    assert new_len.tolist() == [35, 14, 14, 47, -2]
    placed = [0, 1, 2, 3, 4, 5, 6, 10, 11, 15]
    gone = [r for r in range(18) if r not in placed]
    assert torch.equal(qo[placed], q[placed]) and (qo[gone] == 9).all() and (ko[gone] == 9).all()
    written = [(1, 14), (1, 15), (2, 0), (2, 1), (2, 2), (3, 14), (3, 15), (5, 14), (5, 15), (9, 15)]
    for (page, off), r in zip(written, placed):
        assert torch.equal(kp[page, :, off], k[r]) and torch.equal(vp[page, :, off], v[r])
        kp[page, :, off] = 3.0
        vp[page, :, off] = 3.0
    assert (kp == 3).all() and (vp == 3).all()
    with pytest.raises(ValueError, match="page id"):
        paged_append(*args, check=True)
    # a position outside the tables
    cos, sin = tables(8, D, gpu)
    ok = dict(cos=cos.to(gpu), sin=sin.to(gpu))
    with pytest.raises(ValueError, match="position"):
        paged_append(k[:2], v[:2], kp, vp, table[:1].to(gpu), [0], [0, 2], positions=[0, 8], check=True, **ok)
    _, n = paged_append(k[:2], v[:2], kp, vp, table[:1].to(gpu), [0], [0, 2], positions=[-1, 7], **ok)
    assert n.tolist() == [0]


def test_many_ragged_requests_and_inconsistent_offsets(gpu):
    # more requests than a wave looks at; then offsets that decrease
    from cast_amd import paged_append
    rng = np.random.default_rng(1)
    new = rng.integers(0, 4, size=200)
    new[63] = new[64] = 0
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    total = int(cu[-1])
    k = torch.arange(total, device=gpu).float()[:, None, None].expand(total, 1, 8).to(torch.float32).contiguous()
    kp, vp = (torch.full((200, 1, 4, 8), -1.0, device=gpu) for _ in range(2))
    table = torch.arange(200, dtype=torch.int32, device=gpu)[:, None]
    _, n = paged_append(k, k, kp, vp, table, torch.zeros(200, dtype=torch.int32, device=gpu),
                        torch.from_numpy(cu).to(gpu), check=True)
    assert n.tolist() == new.tolist()
    want = torch.full((200, 4), -1.0)
    for b in range(200):
        want[b, :new[b]] = torch.arange(cu[b], cu[b + 1]).float()
    assert torch.equal(kp[:, 0, :, 0].cpu(), want) and torch.equal(vp[:, 0, :, 3].cpu(), want)
    bad = torch.tensor([0, 3, 1, 4], dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError, match="inconsistent"):
        paged_append(k[:4], k[:4], kp, vp, table[:3], [0, 0, 0], bad, check=True)


# ---- together

def test_prompts_then_decode_steps_match_a_dense_cache(gpu):
    """Prompts of three requests into the pages, then steps of append + attention, each step against attention
    over a dense cache of the same rotated keys."""
    from cast_amd import paged_append, paged_attention
    B, Hq, Hkv, D, ps, steps = 3, 8, 2, 64, 16, 20
    g = torch.Generator().manual_seed(11)
    lens = [5, 31, 16]
    width = -(-(max(lens) + steps) // ps)
    table = torch.randperm(B * width, generator=g).to(torch.int32).view(B, width)
    kp, vp = (torch.full((B * width, Hkv, ps, D), float("nan"), dtype=torch.bfloat16, device=gpu) for _ in range(2))
    cos, sin = (x.to(gpu) for x in tables(64, D, gpu))
    draw = lambda n, h: torch.randn((n, h, D), generator=g).to(torch.bfloat16).to(gpu)
    cu = [0] + list(np.cumsum(lens))
    k, v = draw(cu[-1], Hkv), draw(cu[-1], Hkv)
    k_out = torch.empty_like(k)
    _, seq = paged_append(k, v, kp, vp, table.to(gpu), [0] * B, cu, cos=cos, sin=sin, k_out=k_out, check=True)
    dense = [[k_out[cu[b]:cu[b + 1]].cpu(), v[cu[b]:cu[b + 1]].cpu()] for b in range(B)]
    for step in range(steps):
        q, k, v = draw(B, Hq), draw(B, Hkv), draw(B, Hkv)
        ko = torch.empty_like(k)
        qr, seq = paged_append(k, v, kp, vp, table.to(gpu), seq, q=q, cos=cos, sin=sin, k_out=ko)
        out, lse = paged_attention(qr, kp, vp, table.to(gpu), seq, return_lse=True, check=True)
        for b in range(B):
            dense[b] = [torch.cat([x, y[b:b + 1].cpu()]) for x, y in zip(dense[b], (ko, v))]
            n = lens[b] + step + 1
            assert dense[b][0].shape[0] == n == seq[b].item()
            ref = OP.attention(qr[b:b + 1].cpu(), dense[b][0].transpose(0, 1)[None], dense[b][1].transpose(0, 1)[None],
                               [[0]], [n])
            check_attention(out[b:b + 1], lse[b:b + 1], ref, torch.bfloat16, n, D)


def test_unaligned_rows_are_copied_and_kept(gpu):
    # inputs that start off 16 bytes are copied for the call; what the call allocates afterwards must not take the
    # copies' memory
    from cast_amd import paged_append
    g = torch.Generator().manual_seed(0)
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=gpu)
    big = [torch.randn(20 * h * 64 + 1, generator=g).to(torch.bfloat16).to(gpu) for h in (4, 2, 2)]
    q, k, v = (x[1:].view(20, h, 64) for x, h in zip(big, (4, 2, 2)))
    pools = [torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    for _ in range(5):
        out, n = paged_append(k, v, *pools, table, [0], [0, 20], q=q, check=True)
        assert torch.equal(out, q) and n.tolist() == [20]
        for pool, x in zip(pools, (k, v)):
            assert torch.equal(pool.transpose(1, 2).reshape(32, 2, 64)[:20], x)
            pool.zero_()
    with pytest.raises(ValueError, match="aligned"):
        paged_append(k, v, *pools, table, [0], [0, 20], q=q, q_out=q)
    with pytest.raises(ValueError, match="expanded"):
        paged_append(k, v, *pools, table, [0], [0, 20], k_out=torch.zeros((1, 2, 64), dtype=torch.bfloat16,
                                                                          device=gpu).expand(20, 2, 64))


def test_decreasing_offsets_leave_every_length(gpu):
    from cast_amd import paged_append
    k = torch.zeros((4, 1, 64), dtype=torch.bfloat16, device=gpu)
    pools = [torch.zeros((3, 1, 16, 64), dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    table = torch.arange(3, dtype=torch.int32, device=gpu)[:, None]
    cu = torch.tensor([0, 3, 1, 4], dtype=torch.int32, device=gpu)
    _, n = paged_append(k, k, *pools, table, torch.tensor([1, 2, 3], dtype=torch.int32, device=gpu), cu)
    assert n.tolist() == [1, 2, 3]


def test_nothing_to_do(gpu):
    from cast_amd import paged_append, paged_attention
    pools = [torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    none = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device=gpu)
    table = torch.zeros((3, 1), dtype=torch.int32, device=gpu)
    q, n = paged_append(none, none, *pools, table, [4, 5, 6], [0, 0, 0, 0], q=none[:, :, :], check=True)
    assert n.tolist() == [4, 5, 6] and q.shape == (0, 2, 64)
    out, lse = paged_attention(none, *pools, table[:0], torch.zeros(0, dtype=torch.int32, device=gpu), return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)


def test_two_calls_at_once_on_two_streams(gpu):
    # different batches in flight on two streams, each with its own workspace: the bits of the calls alone
    from cast_amd import paged_attention
    sets = []
    for seed, lens in ((1, [4000, 100, 2500]), (2, [700] * 40)):
        kp, vp, table, g = make_cache(gpu, lens, 2, 64, 16, "bf16", seed=seed)
        q = torch.randn((len(lens), 8, 64), generator=g).to(torch.bfloat16)
        sets.append((q.to(gpu), kp.to(gpu), vp.to(gpu), table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu)))
    want = [paged_attention(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(paged_attention(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_the_largest_batch_and_a_tiny_cap(gpu):
    # 65535 requests (one more is refused), and a cap so small that every score is it
    from cast_amd import paged_attention
    B = 65535
    pools = [torch.ones((1, 1, 16, 64), dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    pools[1][0, 0, 1] = 3
    q = torch.ones((B, 1, 64), dtype=torch.bfloat16, device=gpu)
    lens = (torch.arange(B, device=gpu) % 3).to(torch.int32)
    table = torch.zeros((1, 1), dtype=torch.int32, device=gpu).expand(B, 1)
    out = paged_attention(q, *pools, table, lens, check=True)
    assert torch.equal(out[:, 0, 0].float(), torch.tensor([0.0, 1.0, 2.0], device=gpu)[lens.long()])
    from cast_amd._lib import CastError
    with pytest.raises(CastError):
        paged_attention(torch.cat([q, q[:1]]), *pools, table.new_zeros((B + 1, 1)), torch.cat([lens, lens[:1]]))
    out, lse = paged_attention(q[:2] * 0, *pools, table[:2], [2, 2], softcap=1e-45, return_lse=True)
    assert (out == 2).all() and (lse - np.log(2)).abs().max() < 1e-6


def test_empty_tables_strided_workspaces_and_sizes_past_31_bits(gpu):
    from cast_amd import paged_append, paged_attention
    kp, vp, table, g = make_cache(gpu, [300, 17], 2, 64, 16, "bf16")
    kp, vp, table = kp.to(gpu), vp.to(gpu), table.to(gpu)
    lens = torch.tensor([300, 17], dtype=torch.int32, device=gpu)
    q = torch.randn((2, 8, 64), generator=g).bfloat16().to(gpu)
    # tables of no position rotate nothing: not a way to ask for no rotation
    before = kp.clone()
    none = torch.zeros((0, 32), device=gpu)
    with pytest.raises(ValueError, match="no position"):
        paged_append(q[:, :2], q[:, :2], kp, vp, table, lens, cos=none, sin=none)
    assert torch.equal(kp.view(torch.int16), before.view(torch.int16))
    # a workspace whose bytes do not lie side by side
    thin = torch.empty(1, dtype=torch.uint8, device=gpu).expand(1 << 26)
    with pytest.raises(ValueError, match="contiguous"):
        paged_attention(q, kp, vp, table, lens, workspace=thin)
    # a window or split past 31 bits is as good as the largest one
    ref = paged_attention(q, kp, vp, table, lens, kv_split=-1)
    assert torch.equal(paged_attention(q, kp, vp, table, lens, window=(1 << 32) + 5, kv_split=-1), ref)
    assert torch.equal(paged_attention(q, kp, vp, table, lens, kv_split=(1 << 32) + 128), ref)
    assert torch.equal(paged_attention(q, kp, vp, table, lens, kv_split=-(1 << 32) + 128), ref)


@pytest.mark.parametrize("dtype,D,inter", [("bf16", 64, False), ("fp16", 128, True), ("fp32", 40, False)])
def test_two_rows_a_workgroup_are_the_rows_one_by_one(gpu, dtype, D, inter):
    # a call of more rows than the device holds workgroups, an odd number and some behind the last request, against
    # calls of a few requests each: the same bits, in packed and in one-row-each form
    from cast_amd import paged_append
    rng, dt = np.random.default_rng(7), DT[dtype]
    B, ps = 400, 4
    new = rng.integers(0, 13, size=B)
    new[5], new[77], new[78] = 1, 0, 0
    new[-1] += 1 - new.sum() % 2                       # odd
    seq = rng.integers(0, 9, size=B)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    total, tail = int(cu[-1]), 2
    assert total % 2 and total >= 2048
    g = torch.Generator().manual_seed(3)
    k, v, q = (torch.randn((total + tail, h, D), generator=g).to(dt).to(gpu) for h in (1, 1, 2))
    width = int(-(-(seq + new).max() // ps))
    table = torch.randperm(B * width, generator=g).view(B, width).int()
    table[9] = -1                                      # this request has no pages
    new[9] or pytest.fail("the request without pages needs rows")
    table = table.to(gpu)
    cos, sin = (x.to(gpu) for x in tables(64, 32, gpu))
    start = torch.from_numpy(seq.astype(np.int32)).to(gpu)

    def fresh():
        return [torch.full((B * width, 1, ps, D), 5.0, dtype=dt, device=gpu) for _ in range(2)]

    def call(pools, lo, hi, rows, offsets):
        q_out = torch.full_like(q[rows], 7.0)
        _, n = paged_append(k[rows], v[rows], *pools, table[lo:hi], start[lo:hi], offsets, q=q[rows], q_out=q_out, cos=cos,
                            sin=sin, interleaved=inter)
        return q_out, n

    big, small = fresh(), fresh()
    q_big, n_big = call(big, 0, B, slice(0, total + tail), torch.from_numpy(cu).to(gpu))
    parts = []
    for lo in range(0, B, 50):
        rows = slice(int(cu[lo]), int(cu[lo + 50]))
        parts.append(call(small, lo, lo + 50, rows, torch.from_numpy(cu[lo:lo + 51] - cu[lo]).to(gpu)))
    assert torch.equal(q_big[:total], torch.cat([x for x, _ in parts])) and (q_big[total:] == 7).all()
    assert torch.equal(n_big, torch.cat([n for _, n in parts])) and n_big[9] == seq[9]
    assert all(torch.equal(x, y) for x, y in zip(big, small))
    assert (q_big[int(cu[9]):int(cu[10])] == 7).all()
    # one row each, 2401 requests that take turns at the tables' rows
    many = torch.arange(2401, device=gpu) % B
    pools, again = fresh(), fresh()
    lens = (torch.arange(2401, device=gpu) // B).int()             # (rows of one request go to different slots)
    rows = torch.arange(2401, device=gpu) % total
    ks, vs, t = k[rows], v[rows], table[many]
    _, n = paged_append(ks, vs, *pools, t, lens, cos=cos, sin=sin, interleaved=inter)
    for lo in range(0, 2401, 343):
        _, m = paged_append(ks[lo:lo + 343], vs[lo:lo + 343], *again, t[lo:lo + 343], lens[lo:lo + 343], cos=cos, sin=sin,
                            interleaved=inter)
        assert torch.equal(n[lo:lo + 343], m)
    assert all(torch.equal(x, y) for x, y in zip(pools, again))


WIDE = [c for c in CASES if c[9] == 0 and c[7] == 0] + [
    # dtype, Hq, Hkv, D, page size, layout, lengths (window, softcap, kv_split)
    ("bf16", 8, 2, 128, 64, "hnd", [3000, 0, 1, 128, 129, 2048], 0, 0.0, 0),
    ("fp32", 4, 2, 96, 24, "nhd", [1200, 64, 0, 65], 0, 10.0, 0),
    ("fp16", 8, 4, 64, 16, "hnd", [int(x) for x in np.random.default_rng(9).integers(0, 500, 90)], 0, 0.0, 0),
    ("bf16", 4, 4, 256, 32, "hnd", [int(x) for x in np.random.default_rng(8).integers(0, 400, 70)], 0, 0.0, 0),
    ("bf16", 8, 8, 64, 16, "nhd", [int(x) for x in np.random.default_rng(7).integers(0, 300, 110)], 0, 0.0, 0),   # more units than workgroups
    ("fp16", 2, 1, 64, 16, "hnd", [int(x) for x in np.random.default_rng(6).integers(0, 60, 1500)], 0, 0.0, 0),   # lengths past LDS
]


@pytest.mark.parametrize("case", WIDE, ids=lambda c: "-".join(str(x) for x in c[:5]) + f"-b{len(c[6])}")
def test_wide_tables_take_the_schedule_and_narrow_ones_do_not(gpu, case):
    # a unit that may be long is scheduled from the lengths and joined, one that cannot gets a workgroup: both
    # against 64 bits, whatever the tables hold behind the last page
    from cast_amd import paged_attention, paged_workspace_bytes
    dtype, Hq, Hkv, D, ps, layout, lens, _, softcap, _ = case
    print("case wide", case[:6], flush=True)
    kp, vp, table, g = make_cache(gpu, lens, Hkv, D, ps, dtype, layout, seed=len(lens) + D)
    q = torch.randn((len(lens), Hq, D), generator=g).to(DT[dtype])
    ref = OP.attention(q, kp, vp, table, lens, softcap=softcap)
    dev = lambda x: x.to(gpu)
    kd = dev(kp) if layout == "hnd" else dev(kp.transpose(1, 2).contiguous()).transpose(1, 2)
    vd = dev(vp) if layout == "hnd" else dev(vp.transpose(1, 2).contiguous()).transpose(1, 2)
    L = torch.tensor(lens, dtype=torch.int32, device=gpu)
    wide = torch.full((len(lens), (1 << 20) // ps), -9, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    assert paged_workspace_bytes(len(lens), wide.shape[1], ps, Hq, Hkv, D, DT[dtype]) > 0
    for t in (table, wide):
        out, lse = paged_attention(dev(q), kd, vd, dev(t), L, softcap=softcap, return_lse=True, check=True)
        check_attention(out, lse, ref, DT[dtype], max(lens), D)
