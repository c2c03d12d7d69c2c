"""CPU checks of the entry points of beams over a 4-bit cache: invalid arguments are refused before a device is touched, empty
calls are no work, and workspace sizes follow the split."""
import ctypes

import pytest

FAKE = ctypes.c_void_p(4096)    # never dereferenced: validation fails first
ODD = ctypes.c_void_p(4104)     # not 16-byte aligned
BYTE = ctypes.c_void_p(4097)


@pytest.fixture(scope="module")
def lib():
    import forge_amd
    return forge_amd.load()


def call(fn, args, **changed):
    """fn with the named arguments (in order), some of them changed."""
    assert set(changed) <= set(args)
    return fn(*{**args, **changed}.values())


def test_write_and_read(lib):
    w = dict(k=FAKE, v=FAKE, cache=FAKE, slots=FAKE, T=3, Hkv=2, D=64, pages=10, page=16, kt=128, kh=64, vt=128, vh=64, dtype=0,
             stream=None)
    for bad in (dict(k=None), dict(v=None), dict(cache=None), dict(slots=None), dict(D=60), dict(D=264), dict(pages=0), dict(page=8),
                dict(page=24), dict(page=1 << 21), dict(pages=1 << 28), dict(Hkv=65536), dict(kt=12), dict(vh=-8), dict(kt=(1 << 25) + 8), dict(vh=1 << 40), dict(dtype=2),
                dict(dtype=-1), dict(k=ODD), dict(v=ODD), dict(cache=ODD), dict(T=(1 << 31) - 1)):
        assert call(lib.forge_cache4_write, w, **bad) == -1, bad
    for none in (dict(T=0), dict(Hkv=0), dict(D=-8)):
        assert call(lib.forge_cache4_write, dict(w, k=None), **none) == 0, none
    r = dict(cache=FAKE, slots=FAKE, k=FAKE, v=FAKE, T=3, Hkv=2, D=64, pages=10, page=16, dtype=0, stream=None)
    for bad in (dict(k=None), dict(v=None), dict(cache=None), dict(slots=None), dict(D=12), dict(D=264), dict(pages=-1), dict(page=0),
                dict(page=48), dict(dtype=2), dict(k=ODD), dict(cache=ODD)):
        assert call(lib.forge_cache4_read, r, **bad) == -1, bad
    assert call(lib.forge_cache4_read, r, T=0) == 0


def test_attention(lib):
    size = lib.forge_cache4_attention_workspace_size
    a = dict(q=FAKE, cache=FAKE, table=FAKE, lens=FAKE, tree=None, out=FAKE, B=2, T=3, Hq=4, Hkv=2, D=64, pages=100, page=16,
             width=100, scale=0.1, dtype=0, ws=FAKE, bytes=size(2, 3, 4, 2, 64, 1600), stream=None)
    assert a["bytes"] > 0
    for bad in (dict(q=None), dict(cache=None), dict(table=None), dict(lens=None), dict(out=None), dict(T=65), dict(Hkv=3),
                dict(D=12), dict(D=264), dict(pages=0), dict(page=8), dict(page=24), dict(width=0), dict(width=1 << 28),
                dict(pages=1 << 28), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(dtype=2), dict(ws=None),
                dict(bytes=a["bytes"] - 1), dict(cache=ODD), dict(q=ODD), dict(ws=ODD), dict(Hq=1 << 17, Hkv=1)):
        assert call(lib.forge_cache4_attention, a, **bad) == -1, bad
    for none in (dict(B=0), dict(T=0), dict(Hq=0)):
        assert call(lib.forge_cache4_attention, dict(a, q=None), **none) == 0, none


@pytest.mark.parametrize("keys", [(1 << 27) - 2048, (1 << 27) - 1, 1 << 27])
@pytest.mark.parametrize("B", [1, 40])
def test_longest_tables(lib, keys, B):
    """Up to 2^27 positions, in no more chunks than a grid has rows, of no more keys than a chunk's page table has place for:
    16384 where chunks follow the sequences' lengths (an int2 for each comes first then), and 2176 otherwise."""
    row, size = (64 + 2) * 4, lib.forge_cache4_attention_workspace_size(B, 1, 1, 1, 64, keys)
    if B == 1:
        assert (size - 16) % row == 0
        chunks = (size - 16) // row
        assert -(-keys // (chunks - 1)) <= 16384 and 1 < chunks <= 65535
    else:                                                         # 40 2^27 passes what is counted in 32 bits
        assert size % (B * row) == 0
        chunks = size // (B * row)
        assert -(-keys // chunks) <= 2048 + 128 and 1 < chunks <= 65535
    assert lib.forge_cache4_attention_workspace_size(1, 1, 1, 1, 64, (1 << 27) + 1) == 0
    assert lib.forge_cache4_attention_workspace_size(1, 1, 8, 8, 64, 100) == 0     # one chunk


def test_beam_select(lib):
    size = lib.forge_beam_select_workspace_size
    a = dict(logits=FAKE, scores=FAKE, ended=FAKE, end=7, os=FAKE, ob=FAKE, ot=FAKE, B=2, W=3, V=1000, count=6, bs=3000, ws_=1000,
             dtype=0, ws=FAKE, bytes=size(2, 3, 1000, 6), stream=None)
    assert a["bytes"] > 0
    for bad in (dict(logits=None), dict(scores=None), dict(os=None), dict(ob=None), dict(ot=None), dict(ws=None), dict(end=-1),
                dict(end=1000), dict(count=65), dict(W=1025), dict(bs=-1), dict(ws_=-1), dict(dtype=3), dict(dtype=-1), dict(bytes=100),
                dict(ws=ODD), dict(logits=BYTE), dict(logits=ctypes.c_void_p(4098), dtype=2), dict(B=1 << 30, V=1 << 20)):
        assert call(lib.forge_beam_select, a, **bad) == -1, bad
    for none in (dict(B=0), dict(W=0), dict(V=0), dict(count=0)):
        assert call(lib.forge_beam_select, dict(a, logits=None), **none) == 0, none
    assert size(0, 3, 1000, 6) == 0 and size(2, 1025, 1000, 6) == 0 and size(2, 3, 1000, 65) == 0
    assert size(1 << 30, 2, 1 << 20, 1) == 0 and size(1, 1024, 1 << 30, 64) == 0


def test_fork_and_copy(lib):
    import torch
    size = lib.forge_fork_pages_workspace_size(6, 5000)
    assert size == 16 * 6 + 4 * 5 * 1025 and lib.forge_fork_pages_workspace_size(8193, 10) == 0
    at = [ctypes.c_void_p(1 << 20 | i << 16) for i in range(10)]
    a = dict(table=at[0], lens=at[1], parents=at[2], refs=at[3], table_out=at[4], lens_out=at[5], refs_out=at[6], slots=at[7], src=at[8],
             dst=at[9], rows=6, group=3, width=40, pages=5000, page=16, ws=FAKE, bytes=size, stream=None)
    for bad in [{k: None} for k in list(a)[:10]] + [dict(rows=8193, group=1), dict(group=4), dict(group=0), dict(width=0), dict(pages=0),
                                                   dict(page=0), dict(page=24), dict(pages=1 << 28), dict(width=1 << 27), dict(ws=None),
                                                   dict(bytes=size - 1), dict(table_out=at[0]), dict(refs_out=at[3]), dict(lens_out=at[1]),
                                                   dict(refs_out=ctypes.c_void_p(at[3].value + 4000))]:
        assert call(lib.forge_fork_pages, a, **bad) == -1, bad
    assert call(lib.forge_fork_pages, a, rows=0) == 0
    two = (ctypes.c_void_p * 2)(1 << 20, 1 << 21)
    c = dict(caches=ctypes.addressof(two), tensors=2, bytes=4096, pages=10, src=FAKE, dst=FAKE, pairs=3, stream=None)
    for bad in (dict(caches=None), dict(src=None), dict(dst=None), dict(pages=0), dict(bytes=24),
                dict(caches=ctypes.addressof((ctypes.c_void_p * 2)(1 << 20, None))),
                dict(caches=ctypes.addressof((ctypes.c_void_p * 2)(1 << 20, (1 << 21) + 8)))):
        assert call(lib.forge_copy_pages, c, **bad) == -1, bad
    for none in (dict(tensors=0), dict(pairs=0), dict(bytes=0)):
        assert call(lib.forge_copy_pages, c, **none) == 0, none
    assert torch.__version__


def test_operators_refuse():
    """What is not on a device, or no cache, is refused by the operators with an error that says so."""
    import torch
    from forge_amd import ops
    assert ops.cache4_shape(5, 16, 2, 64) == (5, 2, 16, 72) and ops.cache4_shape(1, 32, 1, 200) == (1, 1, 32, 264)
    for D in (0, 12, 264):
        with pytest.raises(ValueError):
            ops.cache4_shape(1, 16, 1, D)
    k = torch.zeros((3, 2, 64), dtype=torch.float16)
    cache = torch.zeros(ops.cache4_shape(5, 16, 2, 64), dtype=torch.uint8)
    slots = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="device"):
        ops.cache4_write(k, k, cache, slots)
    with pytest.raises(TypeError):
        ops.cache4_write(k.float(), k.float(), cache, slots)
    with pytest.raises((ValueError, TypeError)):
        ops.cache4_read(cache, slots, 64)
    with pytest.raises(ValueError, match="device"):
        ops.cache4_attention(torch.zeros((1, 1, 2, 64), dtype=torch.float16), cache, slots[None], slots[:1])
    with pytest.raises(ValueError, match="device"):
        ops.beam_select(torch.zeros((1, 2, 10)), torch.zeros((1, 2)), 2)
    with pytest.raises(TypeError):
        ops.beam_select(torch.zeros((1, 2, 10), dtype=torch.float64), torch.zeros((1, 2)), 2)
    with pytest.raises(ValueError, match="device"):
        ops.fork_pages(slots[None], slots[:1], slots[None, :1], slots, 16)
    with pytest.raises(ValueError, match="device"):
        ops.copy_pages([cache], slots, slots)


def test_beams_host():
    """PagedBeams hands out the prompts' pages, and refuses what does not fit."""
    import torch
    from forge_amd.nn import PagedBeams
    b = PagedBeams(2, 3, 10, 4, 20, "cpu")
    assert b.start([5, 8]).tolist() == [0, 1, 2, 3, 4, 8, 9, 10, 11, 12, 13, 14, 15]
    assert b.table.shape == (6, 6) and b.table[0].tolist() == [0, 1, -1, -1, -1, -1] and b.table[3].tolist() == [2, 3, -1, -1, -1, -1]
    assert b.lens.tolist() == [5, 0, 0, 8, 0, 0] and b.refs.tolist() == [1] * 4 + [0] * 6
    assert b.scores.tolist() == [[0.0, float("-inf"), float("-inf")]] * 2
    assert b.start([0, 1]).tolist() == [0] and b.refs.sum() == 1
    for bad in ([5], [5, -1], [30, 1], [20, 24]):
        with pytest.raises(ValueError):
            b.start(bad)
    with pytest.raises(ValueError):
        PagedBeams(1, 1, 1, 12, 10, "cpu")
    assert torch.equal(b.ended, torch.zeros((2, 3), dtype=torch.bool))
