"""The paged calls straight from tensors: taken for arguments that need no
conversion, with the results of the checked calls, and left to the wrappers
for all others."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def setup(gpu, dtype="bf16", B=3, Hq=8, Hkv=2, D=64, ps=16, pages=40, width=10, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g).to(DT[dtype]).to(gpu)
    table = torch.randperm(pages, generator=g)[:B * width].view(B, width).int().to(gpu)
    s = dict(k=rnd(B, Hkv, D), v=rnd(B, Hkv, D), q=rnd(B, Hq, D), kp=rnd(pages, Hkv, ps, D), vp=rnd(pages, Hkv, ps, D),
             table=table, lens=torch.tensor([5, 130, 77][:B], dtype=torch.int32, device=gpu))
    ang = torch.rand((200, D // 2), generator=g)
    return {**s, "cos": ang.cos().to(gpu), "sin": ang.sin().to(gpu)}


def stream(t):
    from cast_amd import _lib
    return _lib.stream_of(t)


def direct_append(s, **over):
    from cast_amd import _lib
    a = dict(k=s["k"], v=s["v"], kp=s["kp"], vp=s["vp"], table=s["table"], lens=s["lens"], cu=None, q=s["q"], cos=s["cos"],
             sin=s["sin"], pos=None, inter=False, q_out=None, k_out=None, new_len=None)
    a.update(over)
    return _lib.calls().paged_append(*a.values(), stream(s["kp"]))


def direct_attention(s, **over):
    from cast_amd import _lib
    a = dict(q=s["q"], kp=s["kp"], vp=s["vp"], table=s["table"], lens=s["lens"], scale=None, cap=0.0, window=0, split=0,
             lse=False, out=None, ws=None)
    a.update(over)
    return _lib.calls().paged_attention(*a.values(), stream(s["kp"]))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("inter", [False, True])
def test_append_is_the_checked_call(gpu, dtype, inter):
    from cast_amd import paged_append
    one, two = setup(gpu, dtype), setup(gpu, dtype)
    pos = torch.tensor([3, 199, 0], dtype=torch.int32, device=gpu)
    for kw in (dict(), dict(q="q"), dict(q="q", cos="cos", sin="sin", positions=pos), dict(cos="cos", sin="sin")):
        get = lambda s: {n: s[x] if isinstance(x, str) else x for n, x in kw.items()}
        got = paged_append(one["k"], one["v"], one["kp"], one["vp"], one["table"], one["lens"], interleaved=inter, **get(one))
        want = paged_append(two["k"], two["v"], two["kp"], two["vp"], two["table"], two["lens"], interleaved=inter, check=True,
                            **get(two))
        assert (got[0] is None) == (want[0] is None) and (got[0] is None or torch.equal(got[0], want[0]))
        assert torch.equal(got[1], want[1])
        assert torch.equal(one["kp"], two["kp"]) and torch.equal(one["vp"], two["vp"])
    # in place, packed, into the caller's outputs
    cu = torch.tensor([0, 2, 2, 3], dtype=torch.int32, device=gpu)
    outs = []
    for s, check in ((one, False), (two, True)):
        new, k_out = torch.empty_like(s["lens"]), torch.empty_like(s["k"])
        r = paged_append(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["lens"], cu, q=s["q"], cos=s["cos"], sin=s["sin"],
                         q_out=s["q"], k_out=k_out, new_len=new, check=check)
        assert r[0] is s["q"] and r[1] is new
        outs.append((s["q"], k_out, new, s["kp"], s["vp"]))
    assert all(torch.equal(x, y) for x, y in zip(*outs))
    assert direct_append(one) is not None and direct_append(one, q=None, cos=None, sin=None)[0] is None


@pytest.mark.parametrize("dtype", list(DT))
def test_attention_is_the_checked_call(gpu, dtype):
    from cast_amd import paged_attention, paged_workspace_bytes
    s = setup(gpu, dtype)
    args = (s["q"], s["kp"], s["vp"], s["table"], s["lens"])
    space = torch.empty(paged_workspace_bytes(3, 10, 16, 8, 2, 64, DT[dtype]), dtype=torch.uint8, device=gpu)
    for kw in (dict(), dict(softcap=20.0, window=40), dict(kv_split=64), dict(kv_split=-1), dict(sm_scale=0.2),
               dict(workspace=space)):
        got = paged_attention(*args, return_lse=True, **kw)
        want = paged_attention(*args, return_lse=True, check=True, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(paged_attention(*args, **kw), want[0])
    out = torch.empty_like(s["q"])
    assert paged_attention(*args, out=out) is out and torch.equal(out, paged_attention(*args, check=True))
    assert direct_attention(s) is not None


def test_what_needs_a_conversion_or_an_error_is_left_alone(gpu):
    s = setup(gpu)
    before = s["kp"].clone(), s["vp"].clone()
    odd = torch.empty(3 * 2 * 64 + 1, dtype=torch.bfloat16, device=gpu)[1:].view(3, 2, 64)      # 2 bytes off
    common = dict(kp=[s["kp"].cpu(), s["kp"][:0], s["kp"].float(), s["kp"][..., :32], s["kp"].transpose(2, 3), None, 3],
                  table=[s["table"].cpu(), s["table"].long(), s["table"][:, :0], s["table"][0], [[0]], None],
                  lens=[s["lens"].cpu(), s["lens"].long(), s["lens"][:2], [1, 2, 3], torch.stack([s["lens"]] * 2, 1)[:, 0]])
    cases = dict(common, k=[odd, s["k"][:2], s["k"].float(), s["k"].transpose(1, 2), s["k"].cpu()], v=[odd, s["k"][:, :1]],
                 cu=[[0, 1, 2, 3], s["lens"], torch.zeros(4, dtype=torch.int64, device=gpu)],
                 q=[s["q"][:2], s["q"][:, :3], s["q"].float(), s["q"][0]],
                 q_out=[s["q"][:2], s["q"][:1].expand(3, 8, 64), torch.empty_like(s["q"], dtype=torch.float16)],
                 k_out=[odd, s["k"][:, :1].expand(3, 2, 64)], cos=[s["cos"].double(), s["cos"][:0], s["cos"][:, :30], None],
                 pos=[[1, 2, 3], s["lens"].long(), s["lens"][:1]], new_len=[s["lens"].long(), s["lens"][:1]])
    for name, values in cases.items():
        for i, x in enumerate(values):
            assert direct_append(s, **{name: x}) is None, (name, i)
    assert direct_append(s, q=None, q_out=s["q"]) is None
    assert type(direct_append(s, new_len=s["lens"])) is int                 # the library's own refusal
    cases = dict(common, q=[s["q"][:2], s["q"][:, :3], s["q"].float(), s["q"][0], s["q"].cpu()], scale=[1, "x"],
                 cap=[1, -1.0, float("nan"), float("inf")], window=[-1, 1 << 40, 1 << 70, 2.0], split=[-2, 1 << 40, None],
                 out=[s["q"][:2], s["q"][:1].expand(3, 8, 64), torch.empty_like(s["q"], dtype=torch.float16)],
                 ws=[torch.empty(64, dtype=torch.uint8, device=gpu), torch.empty(1 << 24, dtype=torch.uint8),
                     torch.empty(1, dtype=torch.uint8, device=gpu).expand(1 << 24)])
    for name, values in cases.items():
        for i, x in enumerate(values):
            assert direct_attention(s, **{"split": 64, name: x}) is None, (name, i)
    assert type(direct_attention(s, scale=-1.0)) is int
    torch.cuda.synchronize()
    assert torch.equal(s["kp"], before[0]) and torch.equal(s["vp"], before[1])


def test_another_stream_and_a_captured_call(gpu):
    from cast_amd import paged_append, paged_attention
    s, t = setup(gpu), setup(gpu)
    new = torch.empty_like(s["lens"])
    step = lambda x, n, **kw: (paged_append(x["k"], x["v"], x["kp"], x["vp"], x["table"], x["lens"], new_len=n, **kw),
                               paged_attention(x["q"], x["kp"], x["vp"], x["table"], n, **kw))[1]
    want = step(t, torch.empty_like(new), check=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(s, new)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(s, new)
    for i in range(3):
        s["k"].copy_(t["k"].roll(i, 0)), s["q"].mul_(1.5), t["q"].mul_(1.5)
        s["lens"].add_(1), t["lens"].add_(1)
        graph.replay()
        want = step(dict(t, k=t["k"].roll(i, 0)), torch.empty_like(new), check=True)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(s["kp"], t["kp"])


def tree_setup(gpu, dtype="bf16", B=3, Hq=8, Hkv=2, D=64, ps=64, pages=20, width=5, seed=0):
    s = setup(gpu, dtype, B, Hq, Hkv, D, ps, pages, width, seed)
    g = torch.Generator().manual_seed(seed + 1)
    pack = torch.tensor([1, 20, 7][:B])
    total = int(pack.sum())
    rnd = lambda *shape: torch.randn(shape, generator=g).to(DT[dtype]).to(gpu)
    ints = lambda x: torch.as_tensor(x).int().to(gpu)
    words = torch.cat([(1 << torch.arange(1, int(p) + 1)) - 1 for p in pack])      # chains
    return dict(q=rnd(total, Hq, D), kp=s["kp"], vp=s["vp"], table=s["table"], kn=rnd(Hkv, total, D), vn=rnd(Hkv, total, D),
                cu=ints([0, *pack.cumsum(0).tolist()]), pre=ints([200, 0, 131]), pack=ints(pack), mask=words.to(gpu))


def direct_tree(s, **over):
    from cast_amd import _lib
    a = dict(s, scale=None, total_kv=None, lse=False, split=0, out=None, ws=None)
    a.update(over)
    return _lib.calls().paged_tree_attention(*a.values(), stream(s["kp"]))


@pytest.mark.parametrize("dtype", list(DT))
def test_tree_attention_is_the_checked_call(gpu, dtype):
    from cast_amd import paged_tree_attention
    from cast_amd.paged import paged_tree_workspace_bytes
    s = tree_setup(gpu, dtype)
    two = torch.stack([s["mask"], torch.zeros_like(s["mask"])], 1)
    space = torch.empty(paged_tree_workspace_bytes(s["q"], s["kp"], s["table"], 400), dtype=torch.uint8, device=gpu)
    cases = (dict(), dict(total_kv=400), dict(total_kv=400, workspace=space), dict(kv_split=64), dict(sm_scale=0.2),
             dict(kv_split=-1), dict(kv_split=-2), dict(ancestor_mask=two))
    for kw in cases:
        args = dict(zip(("q", "k_pages", "v_pages", "page_table", "k_pack", "v_pack", "cu_q", "prefix_len", "pack_len",
                         "ancestor_mask"), s.values()))
        args.update(kw)
        got = paged_tree_attention(**args, return_lse=True)
        want = paged_tree_attention(**args, return_lse=True, check=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), kw
        assert torch.equal(paged_tree_attention(**args), want[0])
    # (packs as a forward hands them over: token-major, seen head-major)
    kn, vn = (s[x].transpose(0, 1).contiguous().transpose(0, 1) for x in ("kn", "vn"))
    out = torch.empty_like(s["q"])
    assert direct_tree(s, kn=kn, vn=vn, out=out) is out
    assert torch.equal(out, direct_tree(s))


def test_tree_calls_that_need_a_conversion_or_an_error_are_left_alone(gpu):
    s = tree_setup(gpu)
    cases = dict(q=[s["q"][:3], s["q"][:, :3], s["q"].float(), s["q"][0]],
                 kp=[s["kp"].cpu(), s["kp"][:0], s["kp"].float(), s["kp"][:, :, :48], s["kp"][..., :32], None],
                 table=[s["table"].cpu(), s["table"].long(), s["table"][:2], [[0]]],
                 kn=[s["kn"].transpose(0, 1), s["kn"][:, :4], s["kn"].float(), s["kn"].cpu()], vn=[s["vn"][:1]],
                 cu=[s["cu"][:3], s["cu"].long(), s["cu"].cpu(), [0, 1, 21, 28]], pre=[s["pre"].cpu(), [200, 0, 131]],
                 pack=[s["pack"][:2], s["pack"].long()], mask=[s["mask"].int(), s["mask"][:5], s["mask"].cpu(), s["mask"][:, None, None],
                                                               s["mask"][:, None].expand(-1, 3), s["mask"][:, None].expand(-1, 2)],
                 scale=[1, "x"], total_kv=[-1, 1 << 31, 1 << 70, 2.0], split=[None, 1 << 40],
                 out=[s["q"][:3], s["q"][:1].expand(28, 8, 64)],
                 ws=[torch.empty(64, dtype=torch.uint8, device=gpu), torch.empty(1 << 22, dtype=torch.uint8),
                     torch.empty(1, dtype=torch.uint8, device=gpu).expand(1 << 24)])
    for name, values in cases.items():
        for i, x in enumerate(values):
            assert direct_tree(s, **{name: x}) is None, (name, i)
    assert type(direct_tree(s, scale=-1.0)) is int


def test_shared_pages_cut_tables_and_output_over_the_queries(gpu):
    # two requests that share their pages, a table that is some columns of a wider one, results over q: the same bits
    from cast_amd import paged_attention
    for width, split in ((10, 0), (10, 64), (200, 0)):
        s = setup(gpu, pages=40, width=10)
        table = torch.zeros((3, width + 3), dtype=torch.int32, device=gpu)
        table[:, :10] = s["table"]
        table[1, :10] = table[0, :10]
        lens = torch.tensor([130, 130, 77], dtype=torch.int32, device=gpu)
        q = s["q"].clone()
        q[1] = q[0]
        want = paged_attention(q, s["kp"], s["vp"], table[:, :width].contiguous(), lens, kv_split=split)
        assert torch.equal(want[0], want[1])
        assert torch.equal(paged_attention(q, s["kp"], s["vp"], table[:, :width], lens, kv_split=split), want)
        assert paged_attention(q, s["kp"], s["vp"], table[:, :width], lens, kv_split=split, out=q) is q
        assert torch.equal(q, want)


def test_captured_tree_calls_replay_with_new_lengths_and_pages(gpu):
    # two captured calls that share a workspace; lengths, tables and inputs change in place between replays
    from cast_amd import paged_tree_attention
    from cast_amd.paged import paged_tree_workspace_bytes
    sets = [tree_setup(gpu, seed=i) for i in range(2)]
    space = torch.empty(paged_tree_workspace_bytes(sets[0]["q"], sets[0]["kp"], sets[0]["table"], 1000, 64), dtype=torch.uint8,
                        device=gpu)
    call = lambda s, **kw: paged_tree_attention(*s.values(), total_kv=1000, kv_split=64, **kw)
    for s in sets:
        call(s, workspace=space)
    outs, graphs = [torch.empty_like(s["q"]) for s in sets], [torch.cuda.CUDAGraph() for _ in sets]
    for i, s in enumerate(sets):
        with torch.cuda.graph(graphs[i]):
            call(s, out=outs[i], workspace=space)
    for step in range(4):
        for i, s in enumerate(sets):
            s["pre"].copy_(torch.tensor([200 + step, 64 * step, 131 - 3 * step], dtype=torch.int32))
            s["table"].copy_(s["table"].roll(1, 1))
            if step == 2:
                s["table"][2, 0] = -1                       # (rejected in this step alone)
            s["q"].mul_(-1.25)
            want = call(s)
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want), (step, i)
            if step == 2:
                assert (want[21:] == 0).all() and not (want[:21] == 0).all()
                s["table"][2, 0] = 3
        assert not torch.equal(outs[0], outs[1])
