"""CPU-only checks of the operators around the latent paged cache: struct layouts, refusals before any launch."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF = torch.bfloat16


def _layout(struct):
    from dsa_triton_ascend_b200 import _cabi
    cls = getattr(_cabi, struct)
    fields = [n for n, _ in cls._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"dsa_b200.h\"\nint main(){printf(\"%zu\", sizeof(" + struct + "));" + \
        "".join(f'printf(" %zu", offsetof({struct},{n}));' for n in fields) + "return 0;}\n"
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(c, "w").write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe])
        out = [int(v) for v in subprocess.check_output([exe]).split()]
    assert out[0] == ctypes.sizeof(cls)
    assert out[1:] == [getattr(cls, n).offset for n in fields]


@pytest.mark.parametrize("struct", ["DsaRopeParams", "DsaAppendParams", "DsaSpaParams"])
def test_struct_layouts(struct):
    _layout(struct)


FREQ = torch.ones(32)


def _rope(x=None, pos=None, freq=FREQ, **kw):
    from dsa_triton_ascend_b200 import rotary_embedding
    x = torch.zeros(2, 3, 4, 64, dtype=BF) if x is None else x
    pos = torch.zeros(2, 3, dtype=torch.int32) if pos is None else pos
    return rotary_embedding(x, pos, freq, **kw)


@pytest.mark.parametrize("kw", [
    dict(layout="PA_BSND"), dict(layout="TND"), dict(x=torch.zeros(2, 3, 4, 64, dtype=torch.int32)),
    dict(x=torch.zeros(2, 3, 4, 62, dtype=BF)), dict(rotary_offset=2), dict(rotary_offset=-2),
    dict(x=torch.zeros(2, 3, 4, 2048, dtype=BF)), dict(freq=FREQ.double()), dict(freq=FREQ[None]), dict(freq=FREQ[:0]),
    dict(pos=torch.zeros(2, 3)), dict(pos=torch.zeros(2, 4, dtype=torch.int32)), dict(pos=torch.zeros(6, dtype=torch.int32)),
    dict(axis_sections=(16, 16)), dict(axis_sections=(16, 15), pos=torch.zeros(2, 2, 3, dtype=torch.int32)),
    dict(axis_sections=(40, -8), pos=torch.zeros(2, 2, 3, dtype=torch.int32)),
    dict(axis_sections=(8, 8, 8, 4, 4), pos=torch.zeros(5, 2, 3, dtype=torch.int32)),
])
def test_rotary_refusals(kw):
    with pytest.raises(ValueError):
        _rope(**kw)


def test_rotary_refuses_cpu_tensors():
    with pytest.raises(RuntimeError):
        _rope()


def _append(**kw):
    from dsa_triton_ascend_b200 import latent_cache_append
    z = lambda *s: torch.zeros(*s, dtype=BF)
    a = dict(latent=z(2, 3, 1, 512), key_rope=z(2, 3, 1, 64), latent_cache=z(4, 16, 1, 512), rope_cache=z(4, 16, 1, 64),
             inv_freq=FREQ, block_table=torch.zeros(2, 2, dtype=torch.int32), actual_seq_lengths_kv=[3, 3])
    a.update(kw)
    return latent_cache_append(**a)


@pytest.mark.parametrize("kw", [
    dict(layout="PA_BSND"), dict(layout="TND"), dict(latent=torch.zeros(6, 1, 512, dtype=BF), layout="TND"),
    dict(latent=torch.zeros(2, 3, 2, 512, dtype=BF)), dict(latent=torch.zeros(2, 3, 1, 192, dtype=BF)),
    dict(key_rope=torch.zeros(2, 3, 1, 32, dtype=BF)), dict(key_rope=torch.zeros(2, 4, 1, 64, dtype=BF)),
    dict(key_rope=torch.zeros(2, 3, 1, 64, dtype=torch.float16)), dict(rope_cache=torch.zeros(4, 8, 1, 64, dtype=BF)),
    dict(latent_cache=torch.zeros(4, 16, 512, dtype=BF)), dict(latent_cache=torch.zeros(4, 16, 1, 1024, dtype=BF)[..., ::2]),
    dict(latent_cache=torch.zeros(4, 16, 1, 512)), dict(block_table=None), dict(actual_seq_lengths_kv=None),
    dict(index_key=torch.zeros(2, 3, 1, 128, dtype=BF)), dict(index_cache=torch.zeros(4, 16, 1, 128, dtype=BF)),
    dict(index_key=torch.zeros(2, 3, 1, 32, dtype=BF), index_cache=torch.zeros(4, 16, 1, 32, dtype=BF)),
    dict(index_key=torch.zeros(2, 3, 1, 128, dtype=BF), index_cache=torch.zeros(4, 16, 1, 128, dtype=BF), index_rotary_offset=66),
    dict(index_key=torch.zeros(2, 3, 1, 128, dtype=BF), index_cache=torch.zeros(4, 16, 1, 128, dtype=BF), index_rotary_offset=3),
    dict(inv_freq=FREQ[:31]), dict(inv_freq=FREQ.double()), dict(positions=torch.zeros(6, dtype=torch.int32)),
    dict(axis_sections=(16, 16)), dict(positions=torch.zeros(2, 2, 3, dtype=torch.int32)), dict(norm_weight=torch.ones(64)),
    dict(norm_weight=torch.ones(512, dtype=torch.float16)),
])
def test_append_refusals(kw):
    with pytest.raises(ValueError):
        _append(**kw)


def test_append_refuses_cpu_tensors():
    with pytest.raises(RuntimeError):
        _append()


def test_c_interface_refuses_bad_arguments_without_a_gpu():
    from dsa_triton_ascend_b200 import _cabi
    call = lambda f, p: f(ctypes.byref(p), None)
    p = _cabi.DsaRopeParams()
    assert call(_cabi.lib.dsa_rope, p) == -2
    p.struct_size = ctypes.sizeof(p)
    assert call(_cabi.lib.dsa_rope, p) == -1
    p.x = p.positions = p.inv_freq = p.out = 256
    p.batch, p.s1, p.n, p.d, p.pairs, p.axes = 1, 0, 4, 64, 32, 1
    p.sections[0] = 32
    assert call(_cabi.lib.dsa_rope, p) == 0            # no tokens: nothing to launch
    for name, bad in (("pairs", 33), ("pairs", 0), ("offset", 2), ("d", 2048), ("dtype", 3), ("axes", 5), ("axes", 2)):
        old = getattr(p, name)
        setattr(p, name, bad)
        p.sections[1] = 1
        assert call(_cabi.lib.dsa_rope, p) == -3, name
        setattr(p, name, old)
    p.n, p.d = 1 << 20, 1024
    assert call(_cabi.lib.dsa_rope, p) == -8
    a = _cabi.DsaAppendParams()
    assert call(_cabi.lib.dsa_latent_append, a) == -2
    a.struct_size = ctypes.sizeof(a)
    assert call(_cabi.lib.dsa_latent_append, a) == -1
    a.latent = a.key_rope = a.inv_freq = a.seq_k = a.block_table = a.latent_cache = a.rope_cache = 256
    a.batch, a.s1, a.d, a.d_rope, a.block_size, a.max_blocks = 1, 0, 512, 64, 16, 4
    assert call(_cabi.lib.dsa_latent_append, a) == 0
    for name, bad in (("d", 192), ("d_rope", 32), ("dtype", 2), ("block_size", 0), ("latent", 264), ("rope_cache", 258),
                      ("latent_stride_s", 4), ("rope_stride_s", 1), ("layout_q", 2)):
        old = getattr(a, name)
        setattr(a, name, bad)
        assert call(_cabi.lib.dsa_latent_append, a) == -3, name
        setattr(a, name, old)
    a.index_key = 256
    assert call(_cabi.lib.dsa_latent_append, a) == -1
    a.index_cache, a.d_index, a.index_offset = 256, 128, 66
    assert call(_cabi.lib.dsa_latent_append, a) == -3
    a.index_offset, a.max_blocks, a.block_size = 64, 1 << 20, 1 << 12
    assert call(_cabi.lib.dsa_latent_append, a) == -8


def _attend(**kw):
    from dsa_triton_ascend_b200 import shared_prefix_attention
    z = lambda *s: torch.zeros(*s, dtype=BF)
    a = dict(query=z(2, 1, 4, 512), key=z(4, 16, 1, 512), query_rope=z(2, 1, 4, 64), key_rope=z(4, 16, 1, 64),
             block_table=torch.zeros(2, 2, dtype=torch.int32), actual_seq_lengths_kv=[3, 3])
    a.update(kw)
    return shared_prefix_attention(**a)


@pytest.mark.parametrize("kw", [
    dict(sparse_mode=1), dict(query_rope=None), dict(key_rope=None), dict(layout_query="PA_BSND"), dict(layout_query="TND"),
    dict(block_table=None), dict(actual_seq_lengths_kv=None), dict(query=torch.zeros(2, 1, 4, 256, dtype=BF)),
    dict(query=torch.zeros(2, 1, 0, 512, dtype=BF)), dict(query_rope=torch.zeros(2, 1, 4, 32, dtype=BF)),
    dict(query_rope=torch.zeros(2, 1, 3, 64, dtype=BF)), dict(key=torch.zeros(4, 16, 2, 512, dtype=BF)),
    dict(key=torch.zeros(0, 16, 1, 512, dtype=BF)), dict(key=torch.zeros(4, 16, 512, dtype=BF)),
    dict(key_rope=torch.zeros(4, 8, 1, 64, dtype=BF)), dict(key_rope=torch.zeros(4, 16, 1, 64, dtype=torch.float16)),
    dict(block_size=32), dict(shared_prefix_length=-1), dict(shared_prefix_length=torch.zeros(1)),
    dict(shared_prefix_length=torch.zeros(2, dtype=torch.int32)),
])
def test_attention_refusals(kw):
    with pytest.raises(ValueError):
        _attend(**kw)


def test_attention_refuses_cpu_tensors():
    with pytest.raises(RuntimeError):
        _attend()


def test_attention_c_interface_refuses_bad_arguments_without_a_gpu():
    from dsa_triton_ascend_b200 import _cabi
    n, p = ctypes.c_size_t(0), _cabi.DsaSpaParams()
    size = lambda: _cabi.lib.dsa_spa_workspace_bytes(ctypes.byref(p), ctypes.byref(n))
    assert size() == -2
    p.struct_size = ctypes.sizeof(p)
    assert size() == -1
    p.query = p.query_rope = p.key = p.key_rope = p.seq_k = p.block_table = p.out = 256
    p.batch, p.s1, p.n1, p.d, p.d_rope, p.block_size, p.max_blocks, p.key_rows = 2, 1, 4, 512, 64, 16, 2, 64
    assert size() == 0 and n.value >= 256
    for name, bad in (("d", 256), ("d_rope", 0), ("dtype", 2), ("batch", 0), ("n1", 0), ("block_size", 0), ("prefix", -1),
                      ("key_rows", 0), ("sparse_mode", 1), ("kernel", 3), ("key", 264), ("key_rope", 258), ("layout_q", 2)):
        old = getattr(p, name)
        setattr(p, name, bad)
        assert size() == -3, name
        setattr(p, name, old)
    for name, bad in (("max_blocks", 1 << 28), ("s1", 1 << 30)):
        old = getattr(p, name)
        setattr(p, name, bad)
        assert size() == -8, name
        setattr(p, name, old)
    p.layout_q = 1
    assert size() == -1          # TND without cumulative lengths
    p.layout_q, p.return_lse = 0, 1
    assert size() == -1          # statistics asked for, nowhere to put them
    p.return_lse = 0
    assert _cabi.lib.dsa_spa_forward(ctypes.byref(p), None, 0, None) == -4
    assert _cabi.lib.dsa_spa_forward(ctypes.byref(p), 128, 1 << 30, None) == -4
