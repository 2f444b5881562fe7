"""The serving path over pages: the attention hook, the accepted-path append and
ordinary decode steps, as a server runs them, and all of it captured."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(dev, **over):
    transformers = pytest.importorskip("transformers")
    cfg = transformers.Qwen3Config(vocab_size=1024, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                                   num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                                   max_position_embeddings=2048, **over)
    cfg._attn_implementation = "sdpa"
    torch.manual_seed(0)
    model = transformers.Qwen3ForCausalLM(cfg)
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() == 2:
                p.normal_(0.0, 0.06)
    return model.to(dev, torch.bfloat16).eval()


def _pools(gpu, L, n_pages, Hkv, ps, D):
    return [[torch.full((n_pages, Hkv, ps, D), float("nan"), dtype=torch.bfloat16, device=gpu) for _ in range(L)]
            for _ in range(2)]


@torch.inference_mode()
@pytest.mark.parametrize("paged", [True, False], ids=["pages", "store"])
def test_prompt_verify_accept_and_decode_rounds(gpu, paged):
    """Two requests: their prompts' K/V into the cache, a tree verify pass, the accepted rows appended, then three
    ordinary decode steps; logits against the model's own dense cache with plain attention."""
    transformers = pytest.importorskip("transformers")
    import copy
    from cast_amd import greedy_accept, paged_append, serving, tree as T
    from cast_amd.verify import tree_attention_mask
    assert serving.register()
    model = _model(gpu)
    V, L, Hkv, D, ps = 1024, 2, 2, 64, 64
    rng = np.random.default_rng(3)
    prefix, B = [100, 62], 2
    caches = []
    for S in prefix:
        c = transformers.DynamicCache()
        model(torch.from_numpy(rng.integers(0, V, size=S)).to(gpu)[None], past_key_values=c, use_cache=True)
        caches.append(c)
    if paged:
        table = torch.tensor([[5, 1, 7, -1], [2, 6, 0, -1]], dtype=torch.int32, device=gpu)
        buf_k, buf_v = _pools(gpu, L, 8, Hkv, ps, D)
    else:
        table = None
        buf_k, buf_v = _pools(gpu, L, B, Hkv, 4 * ps, D)
    rows = torch.arange(B, dtype=torch.int32, device=gpu)[:, None] if table is None else table
    cu = [0, prefix[0], sum(prefix)]
    for li in range(L):
        kk, vv = (torch.cat([x[0].transpose(0, 1) for x in xs]) for xs in zip(*[(c.layers[li].keys, c.layers[li].values)
                                                                              for c in caches]))
        _, lens = paged_append(kk, vv, buf_k[li], buf_v[li], rows, [0, 0], cu, check=True)
    assert lens.tolist() == prefix

    # ---- a verify pass; the trees' first nodes are what greedy decoding would say, so paths get accepted
    trees, roots = [], []
    for b in range(B):
        top_idx, top_lp = T.block_topk(rng.normal(scale=3.0, size=(15, V)), 8)
        roots.append(int(rng.integers(0, V)))
        trees.append(T.build_tree(top_idx, top_lp, 20))

    def verify():
        kw = {} if table is None else dict(page_table=table)
        ids, pos, cu_q = serving.begin_verify(buf_k, buf_v, prefix, roots, trees, prefix, **kw)
        model.config._attn_implementation = "cast_varlen"
        try:
            out = model(ids, position_ids=pos, past_key_values=transformers.DynamicCache(), use_cache=True).logits[0]
        finally:
            model.config._attn_implementation = "sdpa"
        plan = dict(cu_q=serving.PLAN.cu_q, parent=serving.PLAN.parent)
        serving.PLAN.clear()
        return out, ids[0], cu_q, plan
    logits, _, cu_q, _ = verify()
    for b in range(B):       # put the model's own choice at the root first, to be accepted
        t = trees[b][0]
        trees[b][0] = T.TreeNode(int(logits[cu_q[b]].argmax()), t.depth, t.parent, t.score)
    logits, tok, cu_q, plan = verify()
    for b in range(B):
        nodes = trees[b]
        toks = torch.tensor([[roots[b]] + [nd.token for nd in nodes]], device=gpu)
        p = torch.tensor([[prefix[b]] + [prefix[b] + nd.depth for nd in nodes]], device=gpu)
        want = model(toks, position_ids=p, past_key_values=copy.deepcopy(caches[b]), use_cache=True,
                     attention_mask=tree_attention_mask(prefix[b], nodes, gpu, torch.bfloat16)).logits[0].float()
        err = (logits[cu_q[b]:cu_q[b + 1]].float() - want).abs().max().item()
        assert err <= 2e-2 * want.abs().max().item(), err
    path, plen, bonus, _ = greedy_accept(logits, plan["cu_q"], plan["parent"], tok)
    kw = {} if table is None else dict(page_table=table)
    new_len = serving.append_accepted(buf_k, buf_v, prefix, plan["cu_q"], path, plen, check=True, **kw)
    assert new_len.tolist() == [S + int(n) + 1 for S, n in zip(prefix, plen)] and min(plen.tolist()) >= 1
    for b in range(B):       # the cache now holds the pass's own rows behind the prefix
        keep = [cu_q[b]] + [cu_q[b] + 1 + int(i) for i in path[b, :int(plen[b])]]
        for li in range(L):
            for j, r in enumerate(keep):
                t = prefix[b] + j
                got = buf_k[li][int(rows[b, t // buf_k[li].shape[2]]), :, t % buf_k[li].shape[2]]
                assert torch.equal(got, serving.PACK_KV["k"][li][:, r])

    # ---- ordinary steps, against batch-one decoding over a dense cache of the accepted tokens
    committed = [[roots[b]] + [trees[b][int(i)].token for i in path[b, :int(plen[b])]] for b in range(B)]
    token = bonus
    lens = new_len
    for b in range(B):
        model(torch.tensor([committed[b]], device=gpu), past_key_values=caches[b], use_cache=True)
    for step in range(3):
        ids, pos, after = serving.begin_decode(buf_k, buf_v, lens, token, **kw)
        model.config._attn_implementation = "cast_varlen"
        try:
            got = model(ids, position_ids=pos, past_key_values=transformers.DynamicCache(), use_cache=True).logits[0]
        finally:
            model.config._attn_implementation = "sdpa"
            serving.PLAN.clear()
        assert after.tolist() == [n + 1 for n in lens.tolist()]
        for b in range(B):
            want = model(token[b].view(1, 1), past_key_values=caches[b], use_cache=True).logits[0, -1].float()
            err = (got[b].float() - want).abs().max().item()
            assert err <= 2e-2 * want.abs().max().item(), (step, b, err)
        lens, token = after, got.argmax(-1)


def test_hook_honours_the_forwards_window_and_cap(gpu):
    from cast_amd import paged_attention, serving
    g = torch.Generator().manual_seed(0)
    buf_k, buf_v = ([torch.randn((4, 2, 16, 64), generator=g).to(torch.bfloat16).to(gpu)] for _ in range(2))
    table = torch.tensor([[3, 0], [1, 2]], dtype=torch.int32)
    q, k, v = (torch.randn((1, h, 2, 64), generator=g).to(torch.bfloat16).to(gpu) for h in (4, 2, 2))
    for kw, same in ((dict(softcap=5.0), dict(softcap=5.0)), (dict(sliding_window=7), dict(window=7)),
                     (dict(softcap=None, sliding_window=None), {})):
        _, _, after = serving.begin_decode(buf_k, buf_v, [20, 9], [1, 2], page_table=table)
        out, _ = serving._varlen_attention(None, q, k, v, None, scaling=0.125, **kw)
        serving.PLAN.clear()
        want = paged_attention(q[0].transpose(0, 1), buf_k[0], buf_v[0], table, after, 0.125, **same)
        assert torch.equal(out[0], want)
    with pytest.raises(ValueError, match="no room"):
        serving.begin_decode(buf_k, buf_v, [32, 9], [1, 2], page_table=table)
    with pytest.raises(ValueError, match="row per request"):
        serving.begin_decode(buf_k, buf_v, [20, 9, 1], [1, 2, 3], page_table=table)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_accepted_rows_of_many_layers_match_the_store(gpu, dtype):
    # 70 layers (two launches): the same rows into pages as into a store; a request that passes its table is refused
    from cast_amd import serving
    dt = {"bf16": torch.bfloat16, "fp32": torch.float32}[dtype]
    L, B, Hkv, D, ps = 70, 5, 2, 64, 16
    rng = np.random.default_rng(0)
    lens, packs = [0, 15, 16, 30, 47], [128, 7, 20, 1, 2]
    cu = np.concatenate([[0], np.cumsum(packs)]).astype(np.int32)
    total = int(cu[-1])
    g = torch.Generator().manual_seed(1)
    pk, pv = ([torch.randn((total, Hkv, D), generator=g).to(dt).to(gpu).transpose(0, 1) for _ in range(L)] for _ in range(2))
    path = np.full((B, 128), -1, dtype=np.int32)
    plen = [127, 3, 0, 0, 1]
    for b in range(B):
        path[b, :plen[b]] = np.sort(rng.choice(packs[b] - 1, plen[b], replace=False)) if plen[b] else []
    need = [-(-(n + p + 1) // ps) for n, p in zip(lens, plen)]
    need[4] = 3                                  # 47 + 2 tokens do not fit 3 pages of 16
    table = torch.full((B, max(need)), -1, dtype=torch.int32)
    order = torch.randperm(sum(need), generator=g).to(torch.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    pools = [[torch.full((sum(need), Hkv, ps, D), 2.0, dtype=dt, device=gpu) for _ in range(L)] for _ in range(2)]
    stores = [[torch.full((B, Hkv, 200, D), 2.0, dtype=dt, device=gpu) for _ in range(L)] for _ in range(2)]
    args = (lens, torch.from_numpy(cu).to(gpu), torch.from_numpy(path).to(gpu), torch.tensor(plen, device=gpu), pk, pv)
    got = serving.append_accepted(*pools, *args, page_table=table)
    want = serving.append_accepted(*stores, *args)
    assert got.tolist() == want.tolist()[:4] + [47]
    for pool, store in zip(pools, stores):
        for li in (0, 63, 64, 69):
            for b in range(4):
                n = int(want[b])
                flat = pool[li][table[b, :need[b]].long()].transpose(0, 1).flatten(1, 2)
                assert torch.equal(flat[:, :n], store[li][b, :, :n]) and (flat[:, n:] == 2).all()
    with pytest.raises(ValueError, match="page id|inconsistent"):
        serving.append_accepted(*pools, *args, page_table=table, check=True)


def test_captured_steps_replay_with_new_lengths_pages_and_streams(gpu):
    """Two captured graphs that share one workspace, replayed in turn with lengths and page tables changed in
    place, against eager calls; then the same calls on another stream."""
    from cast_amd import paged_append, paged_attention, paged_workspace_bytes
    B, Hq, Hkv, D, ps, width = 4, 8, 2, 128, 16, 80
    g = torch.Generator(device=gpu).manual_seed(0)
    pools = [torch.randn((B * width, Hkv, ps, D), generator=g, device=gpu).to(torch.bfloat16) for _ in range(2)]
    table = torch.randperm(B * width, generator=g, device=gpu).to(torch.int32).view(B, width)
    lens = torch.tensor([0, 100, 700, 1278], dtype=torch.int32, device=gpu)
    new_len = torch.empty_like(lens)
    q, k, v = (torch.randn((B, h, D), generator=g, device=gpu).to(torch.bfloat16) for h in (Hq, Hkv, Hkv))
    cos, sin = (torch.rand((2048, D // 2), generator=g, device=gpu) for _ in range(2))
    ws = torch.empty(paged_workspace_bytes(B, width, ps, Hq, Hkv, D), dtype=torch.uint8, device=gpu)
    outs = [torch.empty_like(q) for _ in range(2)]
    qr = torch.empty_like(q)

    def step(i):
        paged_append(k, v, *pools, table, lens, q=q, q_out=qr, cos=cos, sin=sin, new_len=new_len)
        paged_attention(qr, *pools, table, new_len, out=outs[i], workspace=ws, softcap=30.0 * i, window=500 * i)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0)
        step(1)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            step(i)
    start = lens.clone()
    for rep in range(5):
        lens.copy_((start * (rep + 1)) // 5)
        table.copy_(torch.randperm(B * width, generator=g, device=gpu).view(B, width))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device=gpu))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (*outs, new_len, qr)]
        kept = [x.clone() for x in pools]
        step(0)
        step(1)
        torch.cuda.synchronize()
        for a, b in zip(got, (*outs, new_len, qr)):
            assert torch.equal(a, b), rep
        assert all(torch.equal(a, b) for a, b in zip(kept, pools))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for x in (*outs, qr):
                x.zero_()
            step(0)
            step(1)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (*outs, new_len, qr)))


def test_no_host_sync_in_a_step(gpu):
    from cast_amd import paged_append, paged_attention, paged_tree_attention
    g = torch.Generator(device=gpu).manual_seed(0)
    pools = [torch.randn((8, 2, 64, 64), generator=g, device=gpu).to(torch.bfloat16) for _ in range(2)]
    table = torch.arange(8, dtype=torch.int32, device=gpu).view(2, 4)
    lens = torch.tensor([70, 3], dtype=torch.int32, device=gpu)
    q, k, v = (torch.randn((2, h, 64), generator=g, device=gpu).to(torch.bfloat16) for h in (4, 2, 2))
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
    one = torch.ones(2, dtype=torch.int32, device=gpu)
    words = torch.ones((2, 2), dtype=torch.int64, device=gpu)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        _, after = paged_append(k, v, *pools, table, lens, q=q)
        a = paged_attention(q, *pools, table, after)
        b = paged_tree_attention(q, *pools, table, k.transpose(0, 1), v.transpose(0, 1), cu, lens, one, words)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    # a pack of the root alone is the token's step: the same numbers but for the order of sums and P's rounding
    # (weights of sum 1, each within 2^-9 of itself, values below 5; then both outputs' half steps)
    assert (a.float() - b.float()).abs().max() <= 5 * 2.0 ** -8 + 2 * 2.0 ** -8 * a.float().abs().max()
