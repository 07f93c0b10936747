"""Refusals and host-side rules of the key/value cache operators.  No GPU: every
check runs before the first CUDA call."""
import ctypes

import pytest
import torch

import q4rdna
from q4rdna import KVAppendArgs, KVAttentionArgs, KVBatchDesc, KVCacheDesc

A = 0x10000  # an aligned address that nothing reads


def desc(**kw):
    d = dict(tiles=A, pages=4, page_tokens=32, kv_heads=2, head_dim=128, format=0)
    d.update(kw)
    return KVCacheDesc(*d.values())


def batch(**kw):
    d = dict(page_table=A, lengths=A, q_start=None, sequences=3, table_stride=2, max_length=0)
    d.update(kw)
    return KVBatchDesc(*d.values())


def append_args(**kw):
    d = dict(type=0, tokens=3, heads=4, k=A, v=A, q=A, q_out=A, k_stride=256, v_stride=256, q_stride=512,
             q_out_stride=512, inv_freq=A, rotary_dim=0, rope=0, positions=None, q_norm=None, k_norm=None,
             norm_eps=1e-6)
    d.update(kw)
    return KVAppendArgs(*d.values())


def attention_args(**kw):
    d = dict(type=0, tokens=3, heads=4, q=A, out=A, q_stride=512, out_stride=512, scale=0.0, window=0)
    d.update(kw)
    return KVAttentionArgs(*d.values())


def refs(*xs):
    return [None if x is None else ctypes.byref(x) for x in xs]


INVALID, SHAPE, ALIGNMENT, WORKSPACE, TOO_LARGE = 1, 2, 3, 4, 11

CACHES = [(dict(tiles=None), INVALID), (dict(tiles=A + 8), ALIGNMENT), (dict(pages=0), INVALID),
          (dict(kv_heads=-1), INVALID), (dict(page_tokens=8), SHAPE), (dict(page_tokens=48), SHAPE),
          (dict(page_tokens=512), SHAPE), (dict(head_dim=96), SHAPE), (dict(head_dim=0), SHAPE),
          (dict(format=2), INVALID)]
BATCHES = [(dict(page_table=None), INVALID), (dict(lengths=None), INVALID), (dict(sequences=-1), INVALID),
           (dict(sequences=2), SHAPE), (dict(table_stride=0), INVALID), (dict(max_length=65), SHAPE),
           (dict(max_length=-1), INVALID)]


@pytest.mark.parametrize("kw,status", CACHES)
def test_cache_refusals(kw, status):
    L = q4rdna.lib
    c, b = refs(desc(**kw), batch())
    assert L.q4rdna_kv_append(c, b, *refs(append_args()), None) == status
    assert L.q4rdna_kv_attention(c, b, *refs(attention_args()), A, 1 << 30, None) == status
    assert L.q4rdna_kv_attention_workspace_bytes(c, b, *refs(attention_args())) == 0
    assert L.q4rdna_kv_dequant(c, A, 1, 0, A, A, None) == status


@pytest.mark.parametrize("kw,status", BATCHES)
def test_batch_refusals(kw, status):
    L = q4rdna.lib
    c, b = refs(desc(), batch(**kw))
    assert L.q4rdna_kv_append(c, b, *refs(append_args()), None) == status
    assert L.q4rdna_kv_attention(c, b, *refs(attention_args()), A, 1 << 30, None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(type=3), INVALID), (dict(heads=-2), INVALID), (dict(rope=2), INVALID), (dict(heads=3), SHAPE),
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(q=None), INVALID), (dict(q_out=None), INVALID),
    (dict(k=A + 4), ALIGNMENT), (dict(q_out=A + 8), ALIGNMENT), (dict(k_stride=255), SHAPE),
    (dict(v_stride=258), ALIGNMENT), (dict(type=1, q_stride=516), ALIGNMENT), (dict(q_stride=511), SHAPE),
    (dict(rotary_dim=24), SHAPE), (dict(rotary_dim=144), SHAPE), (dict(rotary_dim=-16), SHAPE),
    (dict(k_norm=A + 4), ALIGNMENT), (dict(tokens=-1), INVALID), (dict(q_norm=A, norm_eps=-1e-6), INVALID),
    (dict(k_norm=A, norm_eps=float("nan")), INVALID)])
def test_append_refusals(kw, status):
    c, b = refs(desc(), batch())
    assert q4rdna.lib.q4rdna_kv_append(c, b, *refs(append_args(**kw)), None) == status
    assert q4rdna.lib.q4rdna_kv_append(c, b, None, None) == INVALID


@pytest.mark.parametrize("kw,status", [
    (dict(type=-1), INVALID), (dict(heads=0), INVALID), (dict(heads=5), SHAPE), (dict(q=None), INVALID),
    (dict(out=None), INVALID), (dict(out=A + 2), ALIGNMENT), (dict(q_stride=500), SHAPE),
    (dict(out_stride=513), ALIGNMENT), (dict(window=-1), INVALID), (dict(scale=-1.0), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID)])
def test_attention_refusals(kw, status):
    c, b = refs(desc(), batch())
    args = refs(attention_args(**kw))
    assert q4rdna.lib.q4rdna_kv_attention(c, b, *args, A, 1 << 30, None) == status
    assert q4rdna.lib.q4rdna_kv_attention_workspace_bytes(c, b, *args) == 0
    assert q4rdna.lib.q4rdna_kv_attention(c, b, None, A, 1 << 30, None) == INVALID


def test_too_many_rows_are_refused():
    n = (1 << 28) + 1
    c, b = refs(desc(), batch(sequences=n))
    assert q4rdna.lib.q4rdna_kv_append(c, b, *refs(append_args(tokens=n)), None) == TOO_LARGE
    assert q4rdna.lib.q4rdna_kv_attention(c, b, *refs(attention_args(tokens=n)), A, 1 << 40, None) == TOO_LARGE


def test_dequant_refusals():
    c, = refs(desc())
    f = q4rdna.lib.q4rdna_kv_dequant
    assert f(c, A, -1, 0, A, A, None) == INVALID
    assert f(c, A, 1, 3, A, A, None) == INVALID
    assert f(c, None, 1, 0, A, A, None) == INVALID
    assert f(c, A, 1, 0, A + 4, A, None) == ALIGNMENT
    assert f(c, A, 1 << 30, 0, A, A, None) == TOO_LARGE


def test_nothing_to_do_is_ok():
    c, b = refs(desc(), batch(sequences=0))
    none = dict(tokens=0, k=None, v=None, q=None, q_out=None)
    assert q4rdna.lib.q4rdna_kv_append(c, b, *refs(append_args(**none)), None) == 0
    assert q4rdna.lib.q4rdna_kv_attention(c, b, *refs(attention_args(tokens=0, q=None, out=None)), None, 0, None) == 0
    assert q4rdna.lib.q4rdna_kv_dequant(c, None, 0, 0, None, None, None) == 0


def test_sizes():
    assert q4rdna.lib.q4rdna_kv_tile_bytes(128) == 16 + 2 * 16 * 128
    assert q4rdna.lib.q4rdna_kv_tile_bytes(80) == 0
    assert q4rdna.lib.q4rdna_kv_cache_bytes(ctypes.byref(desc())) == 4 * 2 * 2 * (16 + 32 * 128)
    big = desc(pages=1 << 20, page_tokens=256, kv_heads=8)
    assert q4rdna.lib.q4rdna_kv_cache_bytes(ctypes.byref(big)) == (1 << 20) * 8 * 16 * 4112  # past 32 bits


def test_python_refusals():
    cache = q4rdna.KVCache(4, 16, 2, 64, device="cpu")
    assert cache.tiles.shape == (4, 2, 1, 16 + 32 * 64)
    with pytest.raises(ValueError):
        q4rdna.KVCache(4, 24, 2, 64, device="cpu")
    with pytest.raises(ValueError):
        q4rdna.KVCache(4, 16, 2, 64, format=7, device="cpu")
    with pytest.raises(ValueError):
        q4rdna.KVCache(4, 16, 2, 64, tiles=cache.tiles[:3])
    i32 = dict(dtype=torch.int32)
    table, lengths = torch.zeros((3, 2), **i32), torch.zeros(3, **i32)
    for bad in [(table.long(), lengths), (table, lengths.long()), (table[:2], lengths), (table[:, ::2], lengths[:2]),
                (table.expand(3, 2)[:1].expand(3, 2), lengths), (table, lengths, torch.zeros(3, **i32))]:
        with pytest.raises(ValueError):
            q4rdna.KVBatch(*bad)
    wide = torch.zeros((3, 5), **i32)[:, :2]  # rows of a wider table
    rec = q4rdna.KVBatch(wide, lengths)._rec
    assert rec.desc.table_stride == 5 and rec.pages == 2
    with pytest.raises(ValueError):
        q4rdna.KVBatch(table, lengths, max_length=-1)
    x, batch = torch.zeros((3, 2, 64)), q4rdna.KVBatch(table, lengths)
    with pytest.raises(ValueError, match="max_length"):
        q4rdna.kv_attention(cache, q4rdna.KVBatch(table, lengths, max_length=33), x)
    for bad in [x[..., :32], x.transpose(0, 2), x.flatten(), torch.zeros((3, 2, 128))[..., ::2],
                torch.zeros((3, 4, 64))[:, ::2], torch.zeros((3, 100)), x.double(), None, 7, x]:
        with pytest.raises(ValueError):  # the last one for its device
            q4rdna.kv_attention(cache, batch, bad)
        with pytest.raises(ValueError):
            q4rdna.kv_append(cache, batch, bad, x)
        with pytest.raises(ValueError):
            q4rdna.kv_append(cache, batch, x, bad)
    with pytest.raises(ValueError):
        q4rdna.kv_dequant(cache, table)
    with pytest.raises(ValueError):
        q4rdna.kv_dequant(cache, table, dtype="float32")


def test_python_refusals_by_shape_come_before_the_device():
    """Messages name the operand."""
    cache = q4rdna.KVCache(4, 16, 2, 64, device="cpu")
    batch = q4rdna.KVBatch(torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match=r"k is \[rows, heads, 64\]"):
        q4rdna.kv_append(cache, batch, torch.zeros((3, 3, 64)), torch.zeros((3, 2, 64)))
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        q4rdna.kv_attention(cache, batch, torch.zeros((3, 2, 64), dtype=torch.int8))


def test_columns_past_32_bits_are_refused():
    """Rows times query heads of a kv head is an int in the kernels."""
    n, h = 1 << 26, 64
    c, b = refs(desc(kv_heads=1), batch(sequences=n))
    args = dict(tokens=n, heads=h, q_stride=h * 128, out_stride=h * 128)
    assert q4rdna.lib.q4rdna_kv_attention(c, b, *refs(attention_args(**args)), A, 1 << 40, None) == TOO_LARGE
    assert q4rdna.lib.q4rdna_kv_attention_workspace_bytes(c, b, *refs(attention_args(**args))) == 0


def test_an_empty_batch_needs_no_arrays():
    c, b = refs(desc(), batch(page_table=None, lengths=None, sequences=0))
    assert q4rdna.lib.q4rdna_kv_append(c, b, *refs(append_args(tokens=0, k=None, v=None, q=None, q_out=None)), None) == 0
    assert q4rdna.lib.q4rdna_kv_attention(c, b, *refs(attention_args(tokens=0, q=None, out=None)), None, 0, None) == 0


def test_gradients_are_refused():
    """No operator of the cache has a backward pass: a graph that needs one is not cut silently."""
    cache = q4rdna.KVCache(4, 16, 2, 64, device="cpu")
    batch = q4rdna.KVBatch(torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    x, leaf = torch.zeros((3, 2, 64)), torch.zeros((3, 2, 64), requires_grad=True)
    for call in (lambda: q4rdna.kv_attention(cache, batch, leaf), lambda: q4rdna.kv_append(cache, batch, leaf, x),
                 lambda: q4rdna.kv_append(cache, batch, x, leaf)):
        with pytest.raises(ValueError, match="no gradients"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA tensor"):  # goes on to the next check
            call()


def test_tiles_are_read_by_ordinary_loads():
    """The attention is resident while the append before it writes the tiles: nothing is read as data that
    no one writes during the kernel."""
    import os

    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rdna-gfx1201-v0.1_b200", "csrc")
    names = [n for n in os.listdir(csrc) if n.startswith("q4rdna_kv")]
    assert len(names) >= 7
    for n in names:
        with open(os.path.join(csrc, n)) as f:
            text = f.read()
        assert "ld.global.nc" not in text and "__ldg" not in text, n


def test_tangents_are_refused():
    """Forward mode is not cut silently either, under torch.no_grad() neither."""
    import torch.autograd.forward_ad as fwd

    cache = q4rdna.KVCache(4, 16, 2, 64, device="cpu")
    batch = q4rdna.KVBatch(torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    x = torch.zeros((3, 2, 64))
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: q4rdna.kv_attention(cache, batch, dual), lambda: q4rdna.kv_append(cache, batch, dual, x),
                     lambda: q4rdna.kv_append(cache, batch, x, dual)):
            with pytest.raises(ValueError, match="carries a tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="carries a tangent"):
                call()
    with pytest.raises(ValueError, match="CUDA tensor"):
        q4rdna.kv_attention(cache, batch, x)


def test_numbers_past_32_bits_are_refused():
    """The C structures hold 32-bit numbers: a larger one is not taken modulo 2^32."""
    i32 = dict(dtype=torch.int32)
    table, lengths = torch.zeros((3, 2), **i32), torch.zeros(3, **i32)
    assert q4rdna.KVBatch(table, lengths, max_length=1 << 30)._rec.limit == 1 << 30
    for n in ((1 << 30) + 1, 1 << 31, (1 << 32) + 5):
        with pytest.raises(ValueError, match="max_length"):
            q4rdna.KVBatch(table, lengths, max_length=n)
    wide = torch.empty_strided((3, 2), ((1 << 32) + 2, 1), dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="page table"):
        q4rdna.KVBatch(wide, torch.empty(3, dtype=torch.int32, device="meta"))
    tiles = torch.zeros((4, 2, 1, 16 + 32 * 64), dtype=torch.uint8)
    for size in ((4 + (1 << 32), 16, 2, 64), (4 - (1 << 32), 16, 2, 64), (4, 16 + (1 << 32), 2, 64), (4, 16, 2 + (1 << 32), 64),
                 (4, 16, 2, 64 + (1 << 32))):
        with pytest.raises(ValueError):
            q4rdna.KVCache(*size, tiles=tiles)


def test_tiles_cannot_be_replaced():
    """The calls hold the address of the first tiles: with others in their place they would use freed memory."""
    cache = q4rdna.KVCache(4, 16, 2, 64, device="cpu")
    at = cache.tiles.data_ptr()
    with pytest.raises(AttributeError):
        cache.tiles = cache.tiles.clone()
    cache.tiles.fill_(1)
    assert cache.tiles.data_ptr() == at == cache._rec.desc.tiles


def test_a_module_of_another_torch_is_refused(monkeypatch):
    """The call path reads torch's own structures: it runs under the torch that it was built against, or not at all."""
    monkeypatch.setattr(q4rdna, "_kv_module", None)
    monkeypatch.setattr(torch, "__version__", "2.0.0+cu118")
    with pytest.raises(ImportError, match="built against torch"):
        q4rdna._kv()
    monkeypatch.undo()
    assert q4rdna._kv().torch_version == torch.__version__.split("+")[0]


def test_activations_are_read_by_ordinary_loads():
    """The products that overlap the kernel before them (the attention, or their own preparation) read what it wrote."""
    import os
    import re

    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rdna-gfx1201-v0.1_b200", "csrc")
    for n in ("q4rdna_gemv_cta.cuh", "q4rdna_gemv_tc.cuh"):
        with open(os.path.join(csrc, n)) as f:
            text = f.read()
        assert "griddepcontrol.wait" in text
        assert not re.search(r"__ldg\([^;]*T\.x", text) and not re.search(r"__ldg\(fg", text), n
