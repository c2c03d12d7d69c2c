"""CPU checks of the decoder-attention entry points: invalid arguments are refused before a device is touched,
empty calls are no work, and the workspace size follows the split of the keys."""
import ctypes

import pytest

FAKE = ctypes.c_void_p(4096)    # never dereferenced: validation fails first
ODD = ctypes.c_void_p(4104)     # not 16-byte aligned


@pytest.fixture(scope="module")
def lib():
    import forge_amd
    return forge_amd.load()


def call(fn, args, **changed):
    """fn with the named arguments (in order), some of them changed."""
    assert set(changed) <= set(args)
    return fn(*{**args, **changed}.values())


def test_int4(lib):
    quant = dict(w=FAKE, fp16=0, out=FAKE, scale=FAKE, N=4, K=128, group=64, stream=None)
    for bad in (dict(w=None), dict(out=None), dict(scale=None), dict(group=16), dict(group=256), dict(K=96), dict(out=ODD)):
        assert call(lib.forge_quantize_weight_int4, quant, **bad) == -1, bad
    pack = dict(q=FAKE, out=FAKE, N=4, K=128, stream=None)
    for bad in (dict(q=None), dict(out=None), dict(out=ODD), dict(K=40)):
        assert call(lib.forge_pack_weight_int4, pack, **bad) == -1, bad
    lin = dict(x=FAKE, w=FAKE, scale=FAKE, bias=None, out=FAKE, M=2, K=128, N=4, group=128, dtype=0, stream=None)
    for bad in (dict(x=None), dict(w=None), dict(scale=None), dict(out=None), dict(x=ODD), dict(w=ODD), dict(group=48),
                dict(K=192), dict(dtype=2)):
        assert call(lib.forge_int4_linear, lin, **bad) == -1, bad
    for none in (dict(M=0), dict(N=-1), dict(K=0)):
        assert call(lib.forge_int4_linear, dict(lin, x=None), **none) == 0, none


def test_qk_norm_rope(lib):
    a = dict(q=FAKE, k=FAKE, v=FAKE, qw=FAKE, kw=FAKE, cos=FAKE, sin=FAKE, pos=FAKE, q_out=FAKE, k_out=None, kc=FAKE, vc=FAKE,
             slots=FAKE, rows=64, T=2, Hq=4, Hkv=2, D=64, R=64, table=10, qt=256, qh=64, kt=128, kh=64, vt=128, vh=64,
             eps=1e-6, inter=0, dtype=0, stream=None)
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(cos=None), dict(pos=None), dict(q_out=None), dict(vc=None),
                dict(kc=None, vc=None), dict(slots=None), dict(D=60), dict(D=264), dict(R=72), dict(R=24), dict(R=80, D=72),
                dict(table=0), dict(qt=252), dict(kh=-64), dict(dtype=3), dict(qw=ODD), dict(k=ODD), dict(kc=ODD), dict(rows=-1)):
        assert call(lib.forge_qk_norm_rope, a, **bad) == -1, bad
    assert call(lib.forge_qk_norm_rope, a, T=0) == 0


def test_prompt_attention(lib):
    a = dict(q=FAKE, k=FAKE, v=FAKE, cu=FAKE, out=FAKE, n=2, tokens=10, Hq=4, Hkv=2, D=64, qt=256, qh=64, kt=128, kh=64, vt=128,
             vh=64, scale=0.1, causal=1, dtype=0, stream=None)
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(cu=None), dict(out=None), dict(Hkv=3), dict(Hkv=0), dict(D=68),
                dict(D=264), dict(qt=252), dict(vh=-8), dict(kt=1 << 24), dict(scale=0.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(dtype=-1), dict(v=ODD), dict(out=ODD)):
        assert call(lib.forge_prompt_attention, a, **bad) == -1, bad
    for none in (dict(n=0), dict(tokens=0), dict(Hq=0)):
        assert call(lib.forge_prompt_attention, dict(a, q=None), **none) == 0, none


def test_cache_attention(lib):
    size = lib.forge_cache_attention_workspace_size
    a = dict(q=FAKE, k=FAKE, v=FAKE, table=FAKE, lens=FAKE, tree=None, out=FAKE, B=2, T=3, Hq=4, Hkv=2, D=64, pages=100, page=16,
             width=100, scale=0.1, dtype=0, ws=FAKE, bytes=size(2, 3, 4, 2, 64, 1600), stream=None)
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(lens=None), dict(out=None), dict(T=65), dict(Hkv=3),
                dict(D=12), dict(D=264), dict(pages=0), dict(page=0), dict(page=24), dict(width=0), dict(width=1 << 28),
                dict(scale=-1.0), dict(dtype=2), dict(ws=None), dict(bytes=a["bytes"] - 1), dict(k=ODD), dict(ws=ODD)):
        assert call(lib.forge_cache_attention, a, **bad) == -1, bad
    for none in (dict(B=0), dict(T=0), dict(Hq=0)):
        assert call(lib.forge_cache_attention, dict(a, q=None), **none) == 0, none


def test_workspace_size(lib):
    """FP32 sums of D values with a maximum and a sum for each row and chunk, or nothing where one chunk holds all keys."""
    size = lib.forge_cache_attention_workspace_size
    assert size(1, 1, 8, 8, 64, 100) == 0
    assert size(0, 1, 8, 8, 64, 100) == 0 and size(1, 65, 8, 8, 64, 100) == 0 and size(1, 1, 8, 8, 64, 0) == 0
    n = size(2, 3, 8, 2, 128, 5000)
    row = 2 * 3 * 8 * (128 + 2) * 4
    assert n > 0 and n % row == 0 and 2 <= n // row <= (5000 + 127) // 128


def test_tree_masks():
    import torch
    from forge_amd.nn import tree_masks
    got = tree_masks(torch.tensor([[-1, 0, 0, 2], [-1, -1, 1, 1]]))
    assert got.tolist() == [[0b1, 0b11, 0b101, 0b1101], [0b1, 0b10, 0b110, 0b1010]]
    chain = tree_masks(torch.arange(-1, 63)[None])
    assert chain[0, 63] == -1 and chain[0, 62] == (1 << 63) - 1
    for bad in ([[0]], [[-1, 1]], [[-2]]):
        with pytest.raises(ValueError):
            tree_masks(torch.tensor(bad))
    with pytest.raises(ValueError):
        tree_masks(torch.zeros((1, 65), dtype=torch.int64))
