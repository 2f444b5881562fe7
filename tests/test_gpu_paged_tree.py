"""Tree verification over a paged prefix: the same bits as over a store that
holds the same tokens (the same tiles in the same order), and against the
dense oracle in 64 bits.

The 64-bit bound: scores as products of 16-bit elements, exact, in float sums;
P rounded to the operand's 16 bits (a step of 2^-8 in bf16, 2^-11 in fp16 of
each weight, so of sum(weight |v|) <= max |v|), then half a step of the output.
fp32 splits every operand into terms that leave at most 2^-24 of a product.
"""
import math

import numpy as np
import pytest
import torch

from cast_amd import scenarios as SC
from oracle import attn as OA
from oracle import bitmask as OB

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}


def build(gpu, packs, prefix, dtype, Hq, Hkv, D, ps, layout, seed=0, nan_tail=True):
    from cast_amd.tree import TreeNode
    rng = np.random.default_rng(seed)
    trees = []
    for P in packs:
        par = [-1] + [int(rng.integers(0, i)) for i in range(1, P)]
        depth = [0] * P
        for i in range(1, P):
            depth[i] = depth[par[i]] + 1
        trees.append([TreeNode(i, depth[i], par[i] - 1, 0.0) for i in range(1, P)])
    wl = SC._make("paged", trees, prefix, dict(Hq=Hq, Hkv=Hkv, D=D, vocab=1000), dtype, seed, 1.0)
    words = OB.chain_walk_words(wl.packed.parent, wl.cu_q)
    q, k, v = wl.qkv(device="cpu")
    B, cap = len(packs), max(max(prefix), 1)
    ks, vs = (torch.zeros((B, Hkv, cap, D), dtype=q.dtype) for _ in range(2))
    kn, vn = (torch.zeros((Hkv, wl.total_q, D), dtype=q.dtype) for _ in range(2))
    need = [-(-S // ps) for S in prefix]
    order = torch.randperm(sum(need) + 2, generator=torch.Generator().manual_seed(seed)).tolist()
    shape = (len(order), Hkv, ps, D) if layout == "hnd" else (len(order), ps, Hkv, D)
    kp, vp = (torch.full(shape, float("nan"), dtype=q.dtype) for _ in range(2))
    if layout == "nhd":
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    table = torch.full((B, max(need + [1]) + 1), 12345, dtype=torch.int32)
    at = 0
    for b in range(B):
        S, c0, q0 = prefix[b], int(wl.cu_kv[b]), int(wl.cu_q[b])
        for dense, rows, pool in ((ks, k, kp), (vs, v, vp)):
            dense[b, :, :S] = rows[c0:c0 + S].transpose(0, 1)
            for i in range(need[b]):
                n = min(ps, S - i * ps)
                pool[order[at + i], :, :n] = rows[c0 + i * ps:c0 + i * ps + n].transpose(0, 1)
        table[b, :need[b]] = torch.tensor(order[at:at + need[b]], dtype=torch.int32)
        at += need[b]
        for new, rows in ((kn, k), (vn, v)):
            new[:, q0:q0 + packs[b]] = rows[c0 + S:c0 + S + packs[b]].transpose(0, 1)
    pools = [x.to(gpu) if layout == "hnd" else x.transpose(1, 2).contiguous().to(gpu).transpose(1, 2) for x in (kp, vp)]
    dev = [x.to(gpu) for x in (q, ks, vs, kn, vn, table)]
    mask = torch.from_numpy(words.view(np.int64).copy()).to(gpu)
    return wl, words, (q, k, v), dev, pools, mask


CASES = [
    # packs, prefixes, dtype, Hq, Hkv, D, page size, layout, kv_split
    ([1, 2, 63, 64, 65, 128], [64, 1, 63, 65, 300, 1000], "bf16", 8, 2, 128, 64, "hnd", 0),
    ([33, 128, 7], [5000, 129, 64], "bf16", 8, 2, 128, 128, "nhd", 0),
    ([16, 100], [4500, 700], "fp16", 8, 2, 64, 64, "hnd", 256),
    ([16, 100, 1], [700, 0, 192], "fp32", 8, 2, 128, 192, "nhd", 0),
    ([20, 3], [130, 257], "fp32", 4, 1, 64, 64, "hnd", 64),
    ([20, 64], [320, 257], "bf16", 4, 2, 256, 64, "nhd", 0),
    ([20, 64], [320, 257], "fp16", 4, 2, 96, 64, "hnd", 0),
    ([20, 64], [320, 257], "fp32", 4, 2, 80, 128, "hnd", -1),
    ([9] * 70, [int(x) for x in np.random.default_rng(0).integers(0, 300, 70)], "bf16", 4, 2, 128, 64, "hnd", 0),
    ([9, 128], [200, 131], "bf16", 8, 2, 128, 203, "hnd", 0),          # one page per request
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"b{len(c[0])}-{c[2]}-{c[3]}-{c[4]}-d{c[5]}-ps{c[6]}-{c[7]}-s{c[8]}")
def test_same_bits_as_the_store_and_near_64_bits(gpu, case):
    from cast_amd import paged_tree_attention
    from cast_amd.tree_attn import store_tree_attention
    packs, prefix, dtype, Hq, Hkv, D, ps, layout, split = case
    print("case paged tree", case[2:], flush=True)
    wl, words, host, (q, ks, vs, kn, vn, table), (kp, vp), mask = build(gpu, packs, prefix, dtype, Hq, Hkv, D, ps, layout)
    if ps % 64:
        table = table[:, :1].contiguous()
    meta = wl.meta_tensors(gpu)
    total_kv = int(wl.total_kv)
    out, lse = paged_tree_attention(q, kp, vp, table, kn, vn, meta["cu_q"], meta["prefix_len"], meta["pack_len"], mask,
                                    total_kv=total_kv, kv_split=split, return_lse=True, check=True)
    want, wl_lse = store_tree_attention(q, ks, vs, kn, vn, meta["cu_q"], meta["prefix_len"], meta["pack_len"], mask,
                                        total_kv=total_kv, kv_split=split, return_lse=True, check=True)
    assert torch.equal(out, want) and torch.equal(lse, wl_lse)
    q0, k0, v0 = host
    ref, rl = OA.dense_tree_attention(q0, k0, v0, wl.cu_q, wl.cu_kv, wl.prefix_len, wl.pack_len, words,
                                      compute_dtype=torch.float64)
    vmax = float(v0.abs().max())
    score = (D + 8) * 2.0 ** -23 * float((q0.double().abs().amax() * k0.double().abs().amax())) * math.sqrt(D)
    step = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 0.0}[dtype]
    bound = HALF[dtype] * ref.abs() + (step + 2 * score + (max(prefix) + 200) * 2.0 ** -23) * vmax
    assert ((out.double().cpu() - ref).abs() <= bound).all()
    assert ((lse.double().cpu() - rl).abs() <= score + (max(prefix) + 200) * 2.0 ** -23 + 2.0 ** -22 * rl.abs()).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_infinite_values_redo_reads_the_pages_too(gpu, dtype):
    # the padded and fp32 instances compute rows with infinities again from memory: from the pages here
    from cast_amd import paged_tree_attention
    from cast_amd.tree_attn import store_tree_attention
    D = 96 if dtype == "bf16" else 64
    wl, words, host, (q, ks, vs, kn, vn, table), (kp, vp), mask = build(gpu, [5, 40], [300, 150], dtype, 4, 2, D, 64, "hnd")
    vs[0, 1, 130, 7] = float("inf")
    vp[int(table[0, 2]), 1, 2, 7] = float("inf")
    meta = wl.meta_tensors(gpu)
    args = (meta["cu_q"], meta["prefix_len"], meta["pack_len"], mask)
    out = paged_tree_attention(q, kp, vp, table, kn, vn, *args, total_kv=int(wl.total_kv))
    want = store_tree_attention(q, ks, vs, kn, vn, *args, total_kv=int(wl.total_kv))
    assert torch.isinf(out[:5, 2:, 7]).all() and torch.isfinite(out[:, :2]).all()
    assert torch.equal(out, want)


def test_bad_pages_reject_the_request_alone(gpu):
    from cast_amd import paged_tree_attention
    wl, words, host, (q, ks, vs, kn, vn, table), (kp, vp), mask = build(gpu, [5, 40, 9], [300, 150, 700], "bf16", 4, 2,
                                                                         128, 64, "hnd")
    meta = wl.meta_tensors(gpu)
    args = (meta["cu_q"], meta["prefix_len"], meta["pack_len"], mask)
    good, glse = paged_tree_attention(q, kp, vp, table, kn, vn, *args, total_kv=int(wl.total_kv), return_lse=True,
                                      check=True, kv_split=64)
    for bad in (-1, kp.shape[0], 1 << 30):
        t = table.clone()
        t[2, 5] = bad
        out, lse = paged_tree_attention(q, kp, vp, t, kn, vn, *args, total_kv=int(wl.total_kv), return_lse=True,
                                        kv_split=64)
        assert torch.equal(out[:45], good[:45]) and torch.equal(lse[:45], glse[:45])
        assert (out[45:] == 0).all() and torch.isneginf(lse[45:]).all()
        with pytest.raises(ValueError, match="page id"):
            paged_tree_attention(q, kp, vp, t, kn, vn, *args, total_kv=int(wl.total_kv), check=True)
    long = meta["prefix_len"].clone()
    long[1] = table.shape[1] * 64 + 1
    with pytest.raises(ValueError, match="inconsistent"):
        paged_tree_attention(q, kp, vp, table, kn, vn, meta["cu_q"], long, meta["pack_len"], mask, check=True)


def test_offsets_past_32_bits(gpu):
    # pages past 4 GB of the pool
    from cast_amd import paged_tree_attention
    from cast_amd.tree_attn import store_tree_attention
    wl, words, host, (q, ks, vs, kn, vn, table), (kp, vp), mask = build(gpu, [5, 40], [300, 150], "bf16", 4, 2, 128, 64, "hnd")
    n = 90000
    big = torch.empty((2, n, 2, 64, 128), dtype=torch.bfloat16, device=gpu)     # 2.9 GB each
    far = table.clone()
    for b in range(2):
        for i in range(-(-[300, 150][b] // 64)):
            far[b, i] = n - 1 - 10 * b - i
            big[0, n - 1 - 10 * b - i], big[1, n - 1 - 10 * b - i] = kp[table[b, i]], vp[table[b, i]]
    meta = wl.meta_tensors(gpu)
    args = (meta["cu_q"], meta["prefix_len"], meta["pack_len"], mask)
    out = paged_tree_attention(q, big[0], big[1], far, kn, vn, *args, total_kv=int(wl.total_kv), check=True)
    want = store_tree_attention(q, ks, vs, kn, vn, *args, total_kv=int(wl.total_kv))
    assert torch.equal(out, want)
