"""The paged cache's refusals, before any device work (no GPU needed)."""
import pytest
import torch

from cast_amd import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


FAKE = 1 << 20      # never dereferenced: every call here ends before a launch


def append(lib, **over):
    import ctypes
    a = dict(k=FAKE, v=FAKE, kp=FAKE, vp=FAKE, layers=1, table=FAKE, ld=4, max_pages=4, n_pages=8, ps=16, seq=2 * FAKE,
             new=3 * FAKE, B=2, total=2, cu=None, path=None, stride=0, plen=None, q=None, qo=None, ko=None, cos=None,
             sin=None, rope_ld=64, max_pos=100, rot=128, inter=0, pos=None, Hq=8, Hkv=2, D=128, s=[128] * 16, dtype=0,
             status=None, stream=None)
    a.update(over)
    arr = lambda p: None if p is None else (ctypes.c_void_p * max(a["layers"], 1))(*[p or None] * max(a["layers"], 1))
    return lib.cast_paged_append(arr(a["k"]), arr(a["v"]), arr(a["kp"]), arr(a["vp"]), a["layers"], a["table"], a["ld"],
                                 a["max_pages"], a["n_pages"], a["ps"], a["seq"], a["new"], a["B"], a["total"], a["cu"],
                                 a["path"], a["stride"], a["plen"], a["q"], a["qo"], a["ko"], a["cos"], a["sin"],
                                 a["rope_ld"], a["max_pos"], a["rot"], a["inter"], a["pos"], a["Hq"], a["Hkv"], a["D"],
                                 *a["s"], a["dtype"], a["status"], a["stream"])


def test_append_host_validation(lib):
    assert append(lib, B=0) == 0 and append(lib, layers=0) == 0
    assert append(lib, B=-1) == 7 and append(lib, ps=0) == 7 and append(lib, max_pages=-1) == 7
    assert append(lib, dtype=2) == 4 and append(lib, dtype=9) == 4
    assert append(lib, k=None) == 1 and append(lib, seq=None) == 1 and append(lib, table=None) == 1
    assert append(lib, vp=0) == 1                                   # a NULL layer
    assert append(lib, D=100) == 5 and append(lib, D=12, dtype=0) == 5
    assert append(lib, B=3) == 7                                    # one row each, but two rows
    assert append(lib, max_pages=1 << 16, ps=1 << 16) == 7          # slots past 2^31
    assert append(lib, s=[4] + [128] * 15) == 6 and append(lib, k=FAKE + 8) == 6
    assert append(lib, cos=FAKE) == 1 and append(lib, q=FAKE) == 1  # halves of a pair
    assert append(lib, cos=FAKE, sin=FAKE, rot=24) == 5 and append(lib, cos=FAKE, sin=FAKE, rot=144) == 5
    assert append(lib, cos=FAKE + 4, sin=FAKE) == 6 and append(lib, cos=FAKE, sin=FAKE, rope_ld=63) == 7
    assert append(lib, cos=FAKE, sin=FAKE, rope_ld=66) == 6
    assert append(lib, q=FAKE, qo=FAKE, Hq=7) == 2
    # rotation, q and k_out belong to one layer and not to accepted rows
    for extra in (dict(cos=FAKE, sin=FAKE), dict(q=FAKE, qo=FAKE), dict(ko=FAKE)):
        assert append(lib, layers=2, **extra) == 7
        assert append(lib, path=4 * FAKE, plen=5 * FAKE, cu=6 * FAKE, stride=128, **extra) == 7
    assert append(lib, path=4 * FAKE, plen=5 * FAKE, cu=6 * FAKE, stride=127) == 7
    assert append(lib, path=4 * FAKE, plen=5 * FAKE) == 1           # a path needs its packs' offsets


def test_append_refuses_lengths_written_over_its_inputs(lib):
    # workgroups read these while another one writes new_len
    for name in ("seq", "cu", "pos", "table"):
        assert append(lib, **{name: 3 * FAKE}) == _lib.ERR_ALIAS, name
        assert append(lib, **{name: 3 * FAKE - 4}) == _lib.ERR_ALIAS, name
    p = dict(path=4 * FAKE, plen=5 * FAKE, cu=6 * FAKE, stride=128)
    for name in ("path", "plen", "cu"):
        assert append(lib, **{**p, name: 3 * FAKE}) == _lib.ERR_ALIAS, name


def attn(lib, **over):
    a = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, lse=None, table=FAKE, ld=4, max_pages=4, n_pages=8, ps=16, seq=FAKE, B=2,
             Hq=8, Hkv=2, D=128, s=[128] * 10, dtype=0, scale=0.1, cap=0.0, window=0, split=-1, ws=None, wsb=0,
             status=None, stream=None)
    a.update(over)
    return lib.cast_paged_attn_fwd(a["q"], a["k"], a["v"], a["out"], a["lse"], a["table"], a["ld"], a["max_pages"],
                                   a["n_pages"], a["ps"], a["seq"], a["B"], a["Hq"], a["Hkv"], a["D"], *a["s"],
                                   a["dtype"], a["scale"], a["cap"], a["window"], a["split"], a["ws"], a["wsb"],
                                   a["status"], a["stream"])


def test_attention_host_validation(lib):
    assert attn(lib, B=0) == 0
    assert attn(lib, B=-1) == 7 and attn(lib, ps=0) == 7 and attn(lib, window=-1) == 7
    assert attn(lib, B=65536) == 7
    assert attn(lib, Hq=7) == 2 and attn(lib, Hkv=0) == 2
    assert attn(lib, dtype=2) == 4
    for D in (4, 100, 264):
        assert attn(lib, D=D) == 5
    nan = float("nan")
    for bad in (dict(scale=0.0), dict(scale=nan), dict(cap=-1.0), dict(cap=nan), dict(cap=float("inf"))):
        assert attn(lib, **bad) == 9
    assert attn(lib, n_pages=0) == 7 and attn(lib, max_pages=0) == 7    # nothing to read from
    assert attn(lib, max_pages=1 << 16, ps=1 << 15) == 7
    for name in ("q", "k", "v", "out", "table", "seq"):
        assert attn(lib, **{name: None}) == 1, name
    assert attn(lib, s=[128] * 9 + [4]) == 6 and attn(lib, out=FAKE + 2) == 6
    # a call that may split needs its workspace
    need = lib.cast_paged_attn_workspace_size(2, 100, 16, 8, 2, 128, 0, 0, 128)
    assert need > 0 and need % 256 == 0
    assert attn(lib, max_pages=100, split=128) == 1
    assert attn(lib, max_pages=100, split=128, ws=FAKE, wsb=need - 1) == 8
    assert attn(lib, max_pages=100, split=128, ws=FAKE + 16, wsb=need) == 6


def test_workspace_size(lib):
    size = lambda B=2, pages=100, ps=16, Hq=8, Hkv=2, D=128, w=0, dt=0, split=0: lib.cast_paged_attn_workspace_size(
        B, pages, ps, Hq, Hkv, D, w, dt, split)
    assert size() > 0 and size(split=-1) == 0
    assert size(pages=1) == 0                       # too short to split
    assert size(w=1) == 0                           # and so is the window
    assert size(Hq=7) == 0 and size(D=100) == 0 and size(dt=2) == 0 and size(B=0) == 0
    assert size(split=128) > size(split=256) > 0


def test_python_refusals():
    from cast_amd import paged_append, paged_attention
    pool, other = torch.zeros((2, 2, 16, 64)), torch.zeros((2, 2, 16, 32))
    q, table = torch.zeros((1, 4, 64)), torch.zeros((1, 1), dtype=torch.int32)
    with pytest.raises(ValueError, match="page_size"):
        paged_attention(q, pool, other, table, [1])
    with pytest.raises(ValueError, match="on the GPU"):
        paged_attention(q, pool, pool, table, [1])
    with pytest.raises(ValueError, match="on the GPU"):
        paged_append(q, q, pool, pool, table, [0])
    for flag in (_lib.FLAG_BAD_PAGE, _lib.FLAG_BAD_POSITION):
        with pytest.raises(ValueError):
            _lib.raise_device_flags(flag, "x")


def tree(lib, **over):
    a = dict(ptrs=[FAKE] * 3, table=FAKE, ld=4, max_pages=4, n_pages=8, ps=64, more=[FAKE] * 8, words=2, B=1, tq=16, tkv=64,
             Hq=8, Hkv=2, D=128, s=[128] * 14, dtype=0, scale=0.1, split=-1, ws=FAKE, wsb=1 << 20, status=None, stream=None)
    a.update(over)
    return lib.cast_tree_attn_paged_fwd(*a["ptrs"], a["table"], a["ld"], a["max_pages"], a["n_pages"], a["ps"],
                                        *a["more"], a["words"], a["B"], a["tq"], a["tkv"], a["Hq"], a["Hkv"], a["D"],
                                        *a["s"], a["dtype"], a["scale"], a["split"], a["ws"], a["wsb"], a["status"],
                                        a["stream"])


def test_tree_host_validation(lib):
    assert tree(lib, B=0) == 0 and tree(lib, tq=0) == 0
    assert tree(lib, ps=0) == 7 and tree(lib, ps=48) == 7 and tree(lib, max_pages=-1) == 7
    assert tree(lib, max_pages=1 << 20, ps=1 << 12) == 7
    assert tree(lib, Hkv=3) == 2 and tree(lib, dtype=2) == 4 and tree(lib, scale=0.0) == 9 and tree(lib, words=3) == 7
    assert tree(lib, table=None) == 1 and tree(lib, ptrs=[None] * 3) == 1 and tree(lib, more=[None] * 8) == 1
    assert tree(lib, ws=None) == 1 and tree(lib, wsb=255) == 8 and tree(lib, ws=FAKE + 16) == 6
    assert tree(lib, D=12) == 5
    assert tree(lib, s=[128, 128, 4] + [128] * 11) == 6                 # page stride
    # what the scalar kernel takes elsewhere is refused: unaligned strides, rows too far apart
    assert tree(lib, D=96, s=[4] + [128] * 13) == 6
    assert tree(lib, D=96, s=[128] * 4 + [1 << 24] + [128] * 9) == 7
    need = lib.cast_tree_attn_paged_workspace_size(8, 1024, 66560, 32, 8, 128, 0, 64)
    assert need > lib.cast_tree_attn_workspace_size(8, 1024, 66560, 32, 8, 128, 0, 64)
    assert tree(lib, B=8, tq=1024, tkv=66560, Hq=32, Hkv=8, split=64, wsb=need - 1) == 8
    # stream-K has no instances here: sized as unsplit
    assert lib.cast_tree_attn_paged_workspace_size(8, 1024, 66560, 32, 8, 128, 0, -2) == 256


def test_tree_python_refusals():
    from cast_amd import paged_tree_attention
    pool, q = torch.zeros((2, 2, 64, 64)), torch.zeros((4, 4, 64))
    with pytest.raises(ValueError, match="on the GPU"):
        paged_tree_attention(q, pool, pool, torch.zeros((1, 1), dtype=torch.int32), torch.zeros((2, 4, 64)),
                             torch.zeros((2, 4, 64)), [0, 4], [0], [4], torch.zeros(4, dtype=torch.int64))


def test_calls_from_tensors_leave_the_host_to_the_wrappers():
    calls, t = _lib.calls(), torch.zeros((2, 2, 16, 64))
    assert calls.paged_append(*[t] * 15, 0) is None and calls.paged_append(*[None] * 15, 0) is None
    assert calls.paged_attention(*[t] * 12, 0) is None and calls.paged_attention(*[3] * 12, 0) is None
    assert calls.paged_tree_attention(*[t] * 16, 0) is None and calls.paged_tree_attention(*[3] * 16, 0) is None
    for f in (calls.paged_append, calls.paged_attention, calls.paged_tree_attention):
        with pytest.raises(TypeError):
            f(t)
