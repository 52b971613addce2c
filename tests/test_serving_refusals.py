"""What kv_append_rope, attention_shared_prefix and sample_tokens refuse: by shape and type in front of
any device call (CPU tensors, which pass these checks, are refused last), and at the C entries."""
import ctypes as C
import importlib

import pytest
import torch

BF, F8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


def append_args(**kw):
    a = dict(q=torch.zeros(5, 4, 128, dtype=BF), k=torch.zeros(5, 2, 128, dtype=BF), v=torch.zeros(5, 2, 128, dtype=BF),
             cos=torch.zeros(10, 64), sin=torch.zeros(10, 64), positions=torch.zeros(5, dtype=I32),
             K_cache=torch.zeros(3, 16, 2, 128, dtype=BF), V_cache=torch.zeros(3, 16, 2, 128, dtype=BF),
             slots=torch.arange(5))
    a.update(kw)
    return a


def attend_args(**kw):
    a = dict(q=torch.zeros(3, 1, 4, 64, dtype=BF), K_cache=torch.zeros(5, 16, 2, 64, dtype=BF),
             V_cache=torch.zeros(5, 16, 2, 64, dtype=BF), prefix_tables=torch.zeros(1, 2, dtype=I32),
             prefix_lens=torch.zeros(1, dtype=I32), prefix_starts=torch.zeros(2, dtype=I32),
             tables=torch.zeros(3, 2, dtype=I32), lens=torch.zeros(3, dtype=I32))
    a.update(kw)
    return a


def refused(fn, args, error=ValueError, match=None):
    with pytest.raises(error, match=match):
        fn(**args)


Z = torch.zeros
APPEND = [
    (dict(q=Z(5, 4, 64, dtype=BF)), ValueError, "q must be"),
    (dict(k=Z(4, 2, 128, dtype=BF)), ValueError, "q must be"),
    (dict(v=Z(5, 1, 128, dtype=BF)), ValueError, "q must be"),
    (dict(q=Z(5, 4, 128, dtype=torch.float16)), ValueError, "bfloat16 or float32"),
    (dict(q=Z(5, 4, 128)), ValueError, "bfloat16 or float32"),
    (dict(K_cache=Z(3, 16, 1, 128, dtype=BF)), ValueError, "K_cache and V_cache"),
    (dict(K_cache=Z(3, 16, 1, 128, dtype=BF), V_cache=Z(3, 16, 1, 128, dtype=BF)), ValueError, "kv heads"),
    (dict(K_cache=Z(3, 16, 2, 64, dtype=BF), V_cache=Z(3, 16, 2, 64, dtype=BF)), ValueError, "heads of 64"),
    (dict(K_cache=Z(3, 16, 2, 128, dtype=F8)), ValueError, "caches must both"),
    (dict(K_cache=Z(3, 16, 2, 128, dtype=F8), V_cache=Z(3, 16, 2, 128, dtype=F8)), ValueError, "k_scale and v_scale"),
    (dict(K_cache=Z(3, 16, 2, 128, dtype=F8), V_cache=Z(3, 16, 2, 128, dtype=F8), k_scale=Z(1, 1)), ValueError, "k_scale"),
    (dict(k_scale=Z(1, 1), v_scale=Z(1, 1)), ValueError, "k_scale and v_scale"),
    (dict(K_cache=Z(3, 16, 2, 128, dtype=F8), V_cache=Z(3, 16, 2, 128, dtype=F8), k_scale=Z(1), v_scale=Z(1, 1)), ValueError, "PMAX"),
    (dict(q=Z(5, 4, 96, dtype=BF), k=Z(5, 2, 96, dtype=BF), v=Z(5, 2, 96, dtype=BF), K_cache=Z(3, 16, 2, 96, dtype=BF),
          V_cache=Z(3, 16, 2, 96, dtype=BF)), NotImplementedError, "64 or 128"),
    (dict(cos=None), ValueError, "given together"),
    (dict(positions=None), ValueError, "given together"),
    (dict(cos=Z(10, 65), sin=Z(10, 65)), ValueError, "multiple of 8"),
    (dict(cos=Z(10, 68), sin=Z(10, 68)), ValueError, "multiple of 8"),
    (dict(cos=Z(0, 64), sin=Z(0, 64)), ValueError, "cos and sin"),
    (dict(cos=Z(10, 64, dtype=torch.float64)), ValueError, "cos and sin"),
    (dict(sin=Z(9, 64)), ValueError, "cos and sin"),
    (dict(positions=Z(4, dtype=I32)), ValueError, "positions"),
    (dict(positions=Z(5)), ValueError, "positions"),
    (dict(slots=Z(5, dtype=torch.int16)), ValueError, "slots"),
    (dict(slots=Z(5, 1, dtype=I32)), ValueError, "slots"),
    (dict(q_norm=Z(64, dtype=BF)), ValueError, "q_norm"),
    (dict(output=Z(5, 4, 128)), ValueError, "output"),
    (dict(output=Z(5, 4, 64, dtype=BF)), ValueError, "output"),
    (dict(q=3), TypeError, "must be a tensor"),
    (dict(eps="x"), TypeError, "eps"),
    (dict(), ValueError, "CPU tensor"),
]


@pytest.mark.parametrize("i", range(len(APPEND)))
def test_append_refuses(mk, i):
    kw, error, match = APPEND[i]
    refused(mk.kv_append_rope, append_args(**kw), error, match)


ATTEND = [
    (dict(q=Z(3, 9, 4, 64, dtype=BF)), ValueError, "S_tkg"),
    (dict(q=Z(3, 0, 4, 64, dtype=BF)), ValueError, "S_tkg"),
    (dict(q=Z(3, 1, 4, 64)), ValueError, "q must be bfloat16"),
    (dict(q=Z(12, 64, dtype=BF)), ValueError, "q must be bfloat16"),
    (dict(q=Z(3, 1, 5, 64, dtype=BF)), ValueError, "share 2 kv heads"),
    (dict(tables=Z(2, 2, dtype=I32)), ValueError, "tables"),
    (dict(tables=Z(3, 2, dtype=torch.int64)), ValueError, "tables"),
    (dict(lens=Z(3, dtype=torch.int64)), ValueError, "lens"),
    (dict(lens=Z(4, dtype=I32)), ValueError, "lens"),
    (dict(prefix_tables=None), ValueError, "given together"),
    (dict(prefix_starts=Z(1, dtype=I32)), ValueError, "prefix_starts"),
    (dict(prefix_lens=Z(2, dtype=I32)), ValueError, "prefix_lens"),
    (dict(prefix_tables=Z(2, dtype=I32)), ValueError, "prefix_tables"),
    (dict(sink=Z(3)), ValueError, "sink"),
    (dict(output=Z(3, 4, 64, dtype=BF)), ValueError, "output"),
    (dict(K_cache=Z(5, 2, 64, dtype=BF), V_cache=Z(5, 2, 64, dtype=BF)), ValueError, "K_cache and V_cache"),
    (dict(softmax_scale="a"), TypeError, "softmax_scale"),
    (dict(), ValueError, "CPU tensor"),
]


@pytest.mark.parametrize("i", range(len(ATTEND)))
def test_attention_refuses(mk, i):
    kw, error, match = ATTEND[i]
    refused(mk.attention_shared_prefix, attend_args(**kw), error, match)


SAMPLE = [
    (dict(logits=Z(2, 9, dtype=torch.float16)), ValueError, "logits"),
    (dict(logits=Z(9)), ValueError, "logits"),
    (dict(logits=Z(2, 0)), ValueError, "logits"),
    (dict(logits=Z(2, 1).expand(2, (1 << 20) + 1)), ValueError, "logits"),
    (dict(uniforms=Z(3)), ValueError, "uniforms"),
    (dict(uniforms=Z(2, dtype=torch.float64)), ValueError, "uniforms"),
    (dict(temperature=-0.1), ValueError, "temperature"),
    (dict(temperature=float("nan")), ValueError, "temperature"),
    (dict(temperature=Z(3)), ValueError, "temperature"),
    (dict(temperature=Z(2, dtype=I32)), ValueError, "temperature"),
    (dict(top_k=-1), ValueError, "top_k"),
    (dict(top_k=2.5), ValueError, "whole number"),
    (dict(top_k=Z(2)), ValueError, "top_k"),
    (dict(top_p=1.01), ValueError, "top_p"),
    (dict(min_p=2), ValueError, "min_p"),
    (dict(min_p=None), TypeError, "min_p"),
    (dict(output=Z(2, dtype=torch.int64)), ValueError, "output"),
    (dict(output=Z(4, dtype=I32)[::2]), ValueError, "output"),
    (dict(), ValueError, "CPU tensor"),
]


@pytest.mark.parametrize("i", range(len(SAMPLE)))
def test_sample_refuses(mk, i):
    kw, error, match = SAMPLE[i]
    refused(mk.sample_tokens, dict(dict(logits=Z(2, 9), uniforms=Z(2)), **kw), error, match)


@pytest.fixture(scope="module")
def L(mk):
    return importlib.import_module("nki_moe_megakernel_amd._lib")


P = 1 << 20      # an address that no refused call reads


def c_append(L, **kw):
    a = dict(q=P, k=P, v=P, q_stride=(512, 128), k_stride=(256, 128), v_stride=(256, 128), q_out=P, q_out_stride=(512, 128),
             cos=P, sin=P, table_rows=10, rot=128, positions=P, k_cache=P, v_cache=P, k_cache_stride=(4096, 256, 128),
             v_cache_stride=(4096, 256, 128), num_blocks=3, block_len=16, slots=P, T=5, nq=4, nkv=2, d=128)
    a.update(kw)
    return L.load().mkd_kv_append_rope(L.KvAppendArgs(**a), None)


def test_append_c_entry_refuses(L):
    for kw in (dict(T=-1), dict(nq=0), dict(x_dtype=7), dict(rot=4), dict(rot=136), dict(table_rows=0), dict(num_blocks=0),
               dict(num_blocks=1 << 20, block_len=1 << 20), dict(k_cache_stride=(-4096, 256, 128)),
               dict(k_cache_stride=(4096, 257, 128)), dict(q=P + 2), dict(q_stride=(513, 128)), dict(cos=P + 4),
               dict(v_cache=P + 4), dict(T=1 << 30)):
        assert c_append(L, **kw) == L.MKD_ERR_INVALID, kw
    for kw in (dict(q=None), dict(slots=None), dict(sin=None), dict(positions=None), dict(kv_format=1), dict(q_out=None)):
        assert c_append(L, **kw) == L.MKD_ERR_NULL, kw
    assert c_append(L, d=96) == L.MKD_ERR_UNSUPPORTED
    assert c_append(L, kv_format=2) == L.MKD_ERR_UNSUPPORTED
    assert L.load().mkd_kv_append_rope(None, None) == L.MKD_ERR_NULL
    assert c_append(L, T=0, q=None, k=None, v=None, q_out=None, slots=None) == L.MKD_OK


def c_attend(L, ws=P, ws_bytes=1 << 40, **kw):
    a = dict(q=P, q_stride=(256, 256, 64), out=P, out_stride=(256, 256, 64), k_cache=P, v_cache=P,
             k_cache_stride=(2048, 128, 64), v_cache_stride=(2048, 128, 64), num_blocks=5, block_len=16, prefix_tables=P,
             prefix_lens=P, prefix_starts=P, tables=P, lens=P, G=1, prefix_blocks=2, own_blocks=2, softmax_scale=0.1, B=3,
             s_tkg=1, nq=4, nkv=2, d=64)
    a.update(kw)
    return L.load().mkd_attention_shared_prefix(L.SharedPrefixArgs(**a), ws, ws_bytes, None)


def test_attention_c_entry_refuses(L):
    for kw in (dict(B=-1), dict(B=65536), dict(s_tkg=0), dict(s_tkg=9), dict(nq=5), dict(G=-1), dict(G=65536), dict(block_len=0),
               dict(prefix_blocks=1 << 27), dict(own_blocks=1 << 27), dict(num_blocks=0), dict(q=P + 8), dict(q_stride=(257, 256, 64)),
               dict(k_cache=P + 8), dict(k_cache_stride=(2048, 132, 64)), dict(out=P + 2), dict(out_stride=(256, 256, 65))):
        assert c_attend(L, **kw) == L.MKD_ERR_INVALID, kw
    for kw in (dict(q=None), dict(out=None), dict(lens=None), dict(tables=None), dict(prefix_tables=None), dict(prefix_starts=None)):
        assert c_attend(L, **kw) == L.MKD_ERR_NULL, kw
    assert c_attend(L, d=96) == L.MKD_ERR_UNSUPPORTED
    assert c_attend(L, ws_bytes=64, prefix_blocks=200) == L.MKD_ERR_WORKSPACE     # (short contexts need none)
    assert c_attend(L, ws=None, ws_bytes=0, prefix_blocks=200) == L.MKD_ERR_WORKSPACE
    assert L.load().mkd_attention_shared_prefix(None, P, 0, None) == L.MKD_ERR_NULL
    assert c_attend(L, B=0, ws_bytes=0) == L.MKD_OK


def c_sample(L, ws=P, ws_bytes=1 << 40, **kw):
    a = dict(logits=P, row_stride=9, uniforms=P, temperature=1.0, top_p=1.0, tokens=P, B=2, V=9)
    a.update(kw)
    return L.load().mkd_sample_tokens(L.SampleArgs(**a), ws, ws_bytes, None)


def test_sample_c_entry_refuses(L):
    for kw in (dict(B=-1), dict(B=65536), dict(V=0), dict(V=(1 << 20) + 1), dict(logits_dtype=5), dict(row_stride=-9)):
        assert c_sample(L, **kw) == L.MKD_ERR_INVALID, kw
    for kw in (dict(logits=None), dict(uniforms=None), dict(tokens=None), dict(ws=None)):
        assert c_sample(L, **kw) == L.MKD_ERR_NULL, kw
    assert c_sample(L, ws_bytes=100) == L.MKD_ERR_WORKSPACE and c_sample(L, ws=P + 8) == L.MKD_ERR_WORKSPACE
    assert c_sample(L, B=0, logits=None, uniforms=None, tokens=None) == L.MKD_OK
    lib = L.load()
    assert lib.mkd_sample_workspace_bytes(3, 9) > 0 and lib.mkd_sample_workspace_bytes(0, 9) == 0


def test_structs_match_the_header(L):
    """Sizes of the ctypes structs against the header's, through the C compiler's layout rules."""
    import os
    import shutil
    import subprocess
    import tempfile
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with tempfile.TemporaryDirectory() as d:
        src = os.path.join(d, "s.c")
        with open(src, "w") as f:
            f.write('#include <stdio.h>\n#include "mkd.h"\nint main(void){printf("%zu %zu %zu\\n", sizeof(mkd_kv_append_args),'
                    'sizeof(mkd_shared_prefix_args), sizeof(mkd_sample_args));return 0;}\n')
        subprocess.run(["gcc", "-I", os.path.join(root, "include"), src, "-o", os.path.join(d, "s")], check=True)
        sizes = [int(x) for x in subprocess.run([os.path.join(d, "s")], capture_output=True, text=True).stdout.split()]
    assert sizes == [C.sizeof(L.KvAppendArgs), C.sizeof(L.SharedPrefixArgs), C.sizeof(L.SampleArgs)]
