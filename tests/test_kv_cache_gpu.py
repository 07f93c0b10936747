"""The key/value cache operators (q4rdna_kv_append, q4rdna_kv_attention,
q4rdna_kv_dequant) against their definition in 64 bits (tests/kv_reference.py,
where the tolerances are derived).  Needs a B200."""
import math

import pytest
import torch

import kv_reference as ref
import q4rdna
from q4rdna import KV_E4M3, KV_INT8, KVBatch, KVCache, synth

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def make(cuda, seed, lengths, H, D, P, fmt, spare=2, k_scale=1.0):
    """A filled cache (device and CPU tiles) and a shuffled page table; the table's
    places behind a sequence's last page name no page."""
    g = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-n // P) for n in lengths))
    pages = len(lengths) * width + spare
    table = torch.randperm(pages, generator=g)[: len(lengths) * width].reshape(len(lengths), width).int()
    for s, n in enumerate(lengths):
        table[s, -(-n // P):] = 2 ** 31 - 1 if s % 2 else -1
    tiles = torch.empty((pages, H, P // 16, 16 + 32 * D), dtype=torch.uint8).fill_(0xFF)
    ref.fill(tiles, D, fmt, seed, k_scale)
    cache = KVCache(pages, P, H, D, format=fmt, tiles=tiles.to(cuda))
    return cache, tiles, table


def attend(cuda, seed, lengths, news, H, G, D, P, fmt, dtype, window=0, scale=0.0, q_scale=1.5, what=""):
    cache, tiles, table = make(cuda, seed, lengths, H, D, P, fmt)
    T = sum(news)
    starts = [sum(news[:s]) for s in range(len(news) + 1)]
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn((T, H * G, D), generator=g) * q_scale).to(dtype)
    batch = KVBatch(table.to(cuda), i32(lengths, cuda),
                    q_start=None if news == [1] * len(news) else i32(starts, cuda))
    out = q4rdna.kv_attention(cache, batch, q.to(cuda), window=window, scale=scale)
    want = ref.attention(tiles, D, fmt, table, lengths, news, q, window, scale)
    assert out.dtype == dtype and out.shape == q.shape
    assert q4rdna.take_fault() == 0
    assert torch.equal(cache.tiles.cpu(), tiles), "attention wrote the cache"
    return ref.check_attention(out, want, dtype, what)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt", [KV_INT8, KV_E4M3])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_decode(cuda, D, fmt, dtype):
    lengths = [1, 2, 15, 16, 17, 31, 33, 100, 129, 517]
    attend(cuda, 10 + D, lengths, [1] * len(lengths), 2, 4, D, 32, fmt, dtype)


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 9, 16, 17, 24])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_groups(cuda, D, G):
    attend(cuda, 100 + G, [40, 333], [1, 1], 3, G, D, 16, KV_INT8, torch.float32)
    attend(cuda, 200 + G, [65, 18], [3, 2], 1, G, D, 16, KV_E4M3, torch.bfloat16)


@pytest.mark.parametrize("P", [16, 32, 64, 128, 256])
def test_attention_page_sizes(cuda, P):
    attend(cuda, 300 + P, [1, P - 1, P, P + 1, 3 * P + 5], [1] * 5, 2, 4, 128, P, KV_INT8, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [0, 1, 7, 16, 40, 1000])
def test_attention_few_tokens(cuda, window, dtype):
    """Drafts, columns and ragged mixes of prompt pieces and single tokens."""
    attend(cuda, 400 + window, [4, 70, 200, 17], [4, 1, 16, 5], 2, 4, 128, 16, KV_INT8, dtype, window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G,fmt", [(128, 4, KV_E4M3), (128, 4, KV_INT8), (64, 1, KV_INT8), (128, 8, KV_E4M3),
                                     (64, 5, KV_E4M3), (256, 2, KV_INT8), (128, 3, KV_INT8)])
def test_attention_prompts(cuda, D, G, fmt, dtype):
    """Whole prompts and pieces of them beside a single token, lengths that end inside tiles."""
    attend(cuda, 500 + D + G, [300, 129, 77, 513], [300, 100, 1, 250], 2, G, D, 32, fmt, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window", [1, 33, 128, 200])
def test_attention_prompt_windows(cuda, window, dtype):
    attend(cuda, 600 + window, [400, 290], [400, 130], 1, 4, 128, 16, KV_INT8, dtype, window)
    attend(cuda, 700 + window, [400, 290], [200, 290], 2, 2, 64, 64, KV_E4M3, dtype, window)


def test_attention_long(cuda):
    """A long sequence beside short ones: pieces of one row joined, one CTA with several rows."""
    attend(cuda, 800, [20011, 3, 700, 1, 5000, 16], [1] * 6, 2, 4, 128, 64, KV_INT8, torch.float32)
    attend(cuda, 801, [9001, 5], [3, 2], 1, 6, 64, 32, KV_E4M3, torch.float16)
    attend(cuda, 802, [3001], [70], 2, 4, 128, 32, KV_INT8, torch.float32)
    attend(cuda, 803, [3001], [70], 2, 4, 128, 32, KV_E4M3, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths,news,launches", [([400, 6000, 5000, 3], [400, 1, 1, 1], 4), ([6000, 400], [1, 400], 4),
                                                   ([400, 300, 390], [400, 200, 390], 2), ([400, 390], [400, 1], 2)])
def test_attention_prompt_beside_long_decodes(cuda, lengths, news, launches, dtype):
    """Single tokens of long sequences go to the kernel for few columns, beside one prompt too; a few sequences of
    new tokens alone take one kernel."""
    before = q4rdna.launch_count()
    attend(cuda, 805, lengths, news, 2, 4, 128, 16, KV_INT8, dtype)
    assert q4rdna.launch_count() - before == launches


def test_attention_many_sequences(cuda):
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(1, 60, (700,), generator=g).tolist()
    attend(cuda, 810, lengths, [1] * 700, 1, 2, 64, 16, KV_INT8, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S", [31, 32, 33, 64, 65])
def test_attention_batches_about_a_warp(cuda, S, dtype):
    """Sequences of no, one, some and many new tokens side by side."""
    g = torch.Generator().manual_seed(S)
    lengths = torch.randint(40, 300, (S,), generator=g).tolist()
    news = [(1, 0, 3, 40, 1, 1, 2, 1)[(s * 5 + s // 8) % 8] for s in range(S)]
    attend(cuda, 815 + S, lengths, news, 2, 4, 64, 16, KV_INT8, dtype)
    attend(cuda, 817 + S, lengths, [1] * S, 2, 4, 128, 16, KV_E4M3, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths,news", [([7001, 60], [1, 1]), ([4000, 33, 500], [3, 33, 200]), ([2500], [700])])
def test_attention_in_place(cuda, lengths, news, dtype):
    cache, _, table = make(cuda, 825, lengths, 2, 128, 32, KV_INT8)
    start = i32([sum(news[:s]) for s in range(len(news) + 1)], cuda)
    batch = KVBatch(table.to(cuda), i32(lengths, cuda), q_start=None if news == [1, 1] else start)
    q = torch.randn((sum(news), 8, 128), device=cuda).to(dtype)
    want = q4rdna.kv_attention(cache, batch, q)
    got = q4rdna.kv_attention(cache, batch, q, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(q, want)


def test_empty_batch(cuda):
    cache = KVCache(2, 16, 2, 64)
    batch = KVBatch(torch.zeros((0, 3), dtype=torch.int32, device=cuda), i32([], cuda))
    x = torch.zeros((0, 2, 64), device=cuda)
    assert q4rdna.kv_append(cache, batch, x, x, q=x).shape == x.shape
    assert q4rdna.kv_attention(cache, batch, x).shape == x.shape


def test_attention_scores_far_apart(cuda):
    """Scores of hundreds: one token takes all the weight; and a scale of its own."""
    attend(cuda, 820, [333], [1], 2, 4, 128, 16, KV_INT8, torch.float32, q_scale=60.0)
    attend(cuda, 821, [333, 64], [60, 3], 2, 4, 128, 16, KV_E4M3, torch.bfloat16, q_scale=60.0)
    attend(cuda, 822, [333], [2], 2, 4, 128, 16, KV_INT8, torch.float32, scale=0.37)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e37, 1e34, 1e-34, 1e-37])
def test_attention_queries_at_the_ends_of_their_range(cuda, size, dtype):
    """Huge and tiny queries under a scale that brings their scores back."""
    for n in (1, 60):
        attend(cuda, 825, [333], [n], 2, 4, 128, 16, KV_INT8, dtype, q_scale=size, scale=0.1 / size)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("news", [[1, 1, 1, 1], [3, 40, 2, 40]])
def test_attention_empty_rows(cuda, news, dtype):
    """Padded rows (fewer tokens than rows, none at all): zeros, and the others right."""
    attend(cuda, 830, [0, 19, 1, 0], news, 2, 4, 128, 16, KV_INT8, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2, 60])
def test_attention_keeps_other_rows(cuda, n, dtype):
    """Rows before the first and behind the last sequence, and what lies between strided rows."""
    H, G, D, lengths = 2, 4, 128, [60, 61]
    cache, tiles, table = make(cuda, 840, lengths, H, D, 16, KV_INT8)
    T = 3 + 2 * n + 5
    wide = torch.randn((T, H * G * D + 64), device=cuda).to(dtype)
    res = torch.full((T, H * G * D + 32), 7.0, device=cuda, dtype=dtype)
    q, out = wide[:, 64:], res[:, 32:]
    batch = KVBatch(table.to(cuda), i32(lengths, cuda), q_start=i32([3, 3 + n, 3 + 2 * n], cuda))
    got = q4rdna.kv_attention(cache, batch, q, out=out)
    assert got.data_ptr() == out.data_ptr()
    rows = slice(3, 3 + 2 * n)
    want = ref.attention(tiles, D, KV_INT8, table, lengths, [n, n], q.cpu()[rows].unflatten(1, (H * G, D)))
    ref.check_attention(out[rows].unflatten(1, (H * G, D)), want, dtype)
    res[rows, 32:] = 7.0
    assert (res == 7.0).all()


@pytest.mark.parametrize("fmt", [KV_INT8, KV_E4M3])
@pytest.mark.parametrize("news", [[1], [5], [64]])
def test_attention_ignores_what_is_not_seen(cuda, news, fmt):
    """NaN scales, NaN and lowest codes behind the length, before the window and in other pages."""
    H, G, D, P, L, window = 2, 4, 128, 16, 105, 30
    cache, tiles, table = make(cuda, 850, [L], H, D, P, fmt)
    dirty = tiles.clone()
    keep = torch.zeros(tiles.shape[0], dtype=torch.bool)
    n = news[0]
    lo = max(0, L - n - window + 1) // P
    keep[table[0, lo:-(-L // P)].long()] = True
    dirty[~keep] = 0xFF  # NaN scales, code 0xFF (NaN in e4m3)
    _, k, v = ref.parts(dirty, D, fmt)
    last = int(table[0, (L - 1) // P])
    for c in (k, v):
        c.view(torch.uint8)[last, :, (L - 1) % P // 16, L % 16:] = 0x7F if fmt == KV_E4M3 else 0x80
    q = torch.randn((n, H * G, D))
    batch = KVBatch(table.to(cuda), i32([L], cuda), q_start=i32([0, n], cuda))
    out = q4rdna.kv_attention(KVCache(tiles.shape[0], P, H, D, format=fmt, tiles=dirty.to(cuda)), batch, q.to(cuda),
                              window=window)
    ref.check_attention(out, ref.attention(tiles, D, fmt, table, [L], news, q, window), torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_nan_stays_with_its_row(cuda, dtype):
    """A query that is not finite spoils its own row only; a NaN scale the rows that see its tile."""
    H, G, D, n = 1, 2, 64, 40
    cache, tiles, table = make(cuda, 860, [100], H, D, 16, KV_INT8)
    q = torch.randn((n, H * G, D), device=cuda).to(dtype)
    batch = KVBatch(table.to(cuda), i32([100], cuda), q_start=i32([0, n], cuda))
    good = q4rdna.kv_attention(cache, batch, q)
    q[7, 1, 3] = math.nan
    q[9, 0, 5] = math.inf
    out = q4rdna.kv_attention(cache, batch, q)
    bad = torch.zeros((n, H * G), dtype=torch.bool, device=cuda)
    bad[7, 1] = bad[9, 0] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], good[~bad])
    q[7, 1, 3], q[9, 0, 5] = 0.0, 0.0
    good = q4rdna.kv_attention(cache, batch, q)
    cache.tiles.view(torch.float32)[int(table[0, 5]), 0, 0, 1] = math.nan  # value scale of tokens 80..95
    out = q4rdna.kv_attention(cache, batch, q)
    assert torch.isnan(out[20:]).all() and torch.equal(out[:20], good[:20])


def test_attention_values_of_zero_scale(cuda):
    """Tiles stored as zeros (scale 0) count in the softmax."""
    H, G, D = 1, 4, 128
    cache, tiles, table = make(cuda, 870, [90], H, D, 16, KV_INT8)
    for t in (tiles, cache.tiles):
        s, k, v = ref.parts(t, D, KV_INT8)
        for p, z in ((1, 0), (2, 1), (3, 0), (3, 1)):
            s[int(table[0, p]), :, :, z] = 0.0
            (k, v)[z][int(table[0, p])] = 0
    for n in (1, 30):
        q = torch.randn((n, H * G, D))
        batch = KVBatch(table.to(cuda), i32([90], cuda), q_start=i32([0, n], cuda))
        out = q4rdna.kv_attention(cache, batch, q.to(cuda))
        ref.check_attention(out, ref.attention(tiles, D, KV_INT8, table, [90], [n], q), torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,L", [(3, 200), (70, 200), (70, 3001), (40, 40)])
def test_attention_value_scales_far_apart(cuda, n, L, D, dtype):
    """Tiles of tiny, ordinary, huge and no values side by side: each token counts in the softmax by its score alone."""
    H, G, P = 2, 4, 16
    cache, tiles, table = make(cuda, 875, [L], H, D, P, KV_INT8)
    q = torch.randn((n, H * G, D), generator=torch.Generator().manual_seed(2)).to(dtype)
    batch = KVBatch(table.to(cuda), i32([L], cuda), q_start=i32([0, n], cuda))
    blocks = -(-L // P)
    for sizes in ([1e-25, 1e22], [1e22, 1e-25], [0.0, 1e10], [1e30, 0.0, 1.0, 1e-20], [1.0, 1e-28, 0.0]):
        t = tiles.clone()
        s, _, v = ref.parts(t, D, KV_INT8)
        i = torch.arange(blocks)
        by = torch.tensor(sizes)[i * len(sizes) // blocks if L < 1000 else i % len(sizes)]
        pages = table[0, :blocks].long()
        s[pages, :, 0, 1] *= by[:, None]
        v[pages[by == 0]] = 0  # a tile of scale 0 is stored as zeros
        cache.tiles.copy_(t)
        out = q4rdna.kv_attention(cache, batch, q.to(cuda))
        want, mag, big = ref.attention(t, D, KV_INT8, table, [L], [n], q)
        # Bounds relative to the row's largest sum p |v|, not each element's.  w sv, the weight times the value's scale, is
        # held relative to the row's largest one, W (as p >= 2^7 for W itself, in two f16 terms whose last bit is 2^-24):
        # a term is off by 2^-25 / 2^7 W at most, times a code 2^-25 W, L terms by L 2^-25 W, where an element with
        # code 0 under W may be 2^-150 W.  The row's largest sum is at least W times its token's largest code, over 2^4: L
        # 2^-29 = 2^-17.4 relative at 3001, under the 2 A 2^-19 >= 2^-16 of the bound (A >= 4 here; asserted).
        assert L * 2.0 ** -29 <= 2 * big[-1].min() * 2.0 ** -19
        ref.check_attention(out, (want, mag.amax(-1, keepdim=True), big), dtype, f"{sizes}")


def test_bad_metadata_sets_the_fault(cuda):
    """Pages outside the cache, lengths above the bound and q_start outside the
    rows are refused on the device: bit 3, nothing read or written there."""
    H, G, D, P = 2, 4, 64, 16
    cache, tiles, table = make(cuda, 880, [40, 40], H, D, P, KV_INT8)
    q = torch.randn((2, H * G, D), device=cuda)
    k = torch.randn((2, H, D), device=cuda)
    good = {n: q4rdna.kv_attention(cache, KVBatch(table.to(cuda), i32([40, 40], cuda), q_start=start), q)
            for n, start in ((False, None), (True, i32([0, 1, 2], cuda)))}  # a kernel each
    assert q4rdna.take_fault() == 0
    bad = table.clone()
    bad[1, 1] = tiles.shape[0]
    for t, lengths, start in [(bad, [40, 40], None), (table, [40, 49], None), (table, [40, -3], None),
                              (table, [40, 40], [0, 1, 3]), (table, [40, 40], [0, 1, 0])]:
        batch = KVBatch(t.to(cuda), i32(lengths, cuda), q_start=None if start is None else i32(start, cuda))
        out = q4rdna.kv_attention(cache, batch, q)
        assert torch.equal(out[0], good[start is not None][0])
        assert q4rdna.take_fault() == 8
    # the append with the same tables: the other sequence's row is written, nothing else
    for t, lengths in [(bad.roll(0), [33, 17]), (table, [33, 49])]:
        before = cache.tiles.clone()
        q4rdna.kv_append(cache, KVBatch(t.to(cuda), i32(lengths, cuda)), k, k)
        assert q4rdna.take_fault() == 8
        changed = (cache.tiles != before).flatten(1).any(1).nonzero().flatten().tolist()
        assert changed in ([int(table[0, 2])], [])
    bad = i32([-1, tiles.shape[0], int(table[0, 0])], cuda)
    kk, vv = q4rdna.kv_dequant(cache, bad)
    assert q4rdna.take_fault() == 8
    assert not kk[:2].any() and not vv[:2].any() and kk[2].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [2, 45])
def test_attention_without_a_page(cuda, n, D, dtype):
    """Tokens on a page outside the cache are not seen, whichever kernel the columns choose; the other sequence is right."""
    H, G, P, L = 2, 4, 32, 200
    cache, tiles, table = make(cuda, 885, [L, L], H, D, P, KV_INT8)
    q = torch.randn((2 * n, H * G, D), generator=torch.Generator().manual_seed(1)).to(dtype)
    start = i32([0, n, 2 * n], cuda)
    for missing in ([2], [0, 1, 2, 3], [4, 6], list(range(7))):
        bad = table.clone()
        bad[1, missing] = torch.tensor([tiles.shape[0], -1, 2 ** 31 - 1] * 3)[: len(missing)].int()
        batch = KVBatch(bad.to(cuda), i32([L, L], cuda), q_start=start)
        out = q4rdna.kv_attention(cache, batch, q.to(cuda))
        assert q4rdna.take_fault() == 8
        ref.check_attention(out[:n], ref.attention(tiles, D, KV_INT8, table, [L], [n], q[:n]), dtype, "other sequence")
        kk, vv = (x[table[1, :7].long()].transpose(0, 1).flatten(1, 2)[:, :L] for x in ref.numbers(tiles, D, KV_INT8))
        there = torch.tensor([t // P not in missing for t in range(L)])
        want = [torch.zeros((n, H * G, D), dtype=torch.float64) for _ in range(3)]
        for i in range(n):
            at = there.clone()
            at[L - n + i + 1:] = False
            if not at.any():
                continue
            x = q[n + i].double().reshape(H, G, D)
            w = torch.softmax(x @ kk[:, at].transpose(-1, -2) / math.sqrt(D), -1)
            want[0][i], want[1][i] = ((w @ v).reshape(H * G, D) for v in (vv[:, at], vv[:, at].abs()))
            want[2][i] = ((x.abs() @ kk[:, at].abs().transpose(-1, -2)) / math.sqrt(D)).amax(-1).reshape(H * G, 1)
        ref.check_attention(out[n:], want, dtype, f"without {missing}")


def test_append_beside_bad_metadata(cuda):
    """The other sequence's row is written, each time anew, and nothing else."""
    H, D, P = 2, 64, 16
    cache, tiles, table = make(cuda, 890, [40, 40], H, D, P, KV_INT8)
    bad = table.clone()
    bad[1, 1] = tiles.shape[0]
    for i, (t, lengths) in enumerate([(bad, [33, 17]), (table, [34, 49]), (table, [35, -1])]):
        k = torch.randn((2, H, D), generator=torch.Generator().manual_seed(i))
        before = cache.tiles.cpu()
        q4rdna.kv_append(cache, KVBatch(t.to(cuda), i32(lengths, cuda)), k.to(cuda), k.to(cuda))
        assert q4rdna.take_fault() == 8
        after = cache.tiles.cpu()
        changed = (after != before).flatten(1).any(1).nonzero().flatten().tolist()
        assert changed == [int(table[0, 2])]
        ref.check_append(before, after, D, KV_INT8, table, lengths[:1], [1], k[:1].double(), k[:1].double())


def test_pages_past_32_bits(cuda):
    """A cache above 4 GiB: tokens in its last pages."""
    H, D, P, L = 8, 128, 256, 300
    per = H * (P // 16) * (16 + 32 * D)
    pages = (1 << 32) // per + 3
    cache = KVCache(pages, P, H, D)
    table = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32)
    k, v, q = (torch.randn((L, H, D), device=cuda) for _ in range(3))
    batch = KVBatch(table.to(cuda), i32([L], cuda), q_start=i32([0, L], cuda))
    q4rdna.kv_append(cache, batch, k, v)
    small = torch.cat((torch.zeros_like(cache.tiles[:1]), cache.tiles[-2:])).cpu()
    ref.check_append(torch.zeros_like(small), small, D, KV_INT8, table - (pages - 3), [L], [L], k.double().cpu(),
                     v.double().cpu())
    assert not cache.tiles[: 2 ** 32 // per - 1].any()
    for rows in (slice(L - 1, L), slice(0, L)):
        n = q[rows].shape[0]
        out = q4rdna.kv_attention(cache, KVBatch(table.to(cuda), i32([L], cuda), q_start=i32([0, n], cuda)), q[rows])
        ref.check_attention(out, ref.attention(small, D, KV_INT8, table - (pages - 3), [L], [n], q[rows].cpu()),
                            torch.float32)


# ------------------------------------------------------------------ append

def run_append(cuda, seed, lengths, news, H, G, D, P, fmt, dtype, neox=True, rot=None, norm=True, positions=None,
               x_scale=1.0, in_place=False):
    cache, tiles, table = make(cuda, seed, lengths, H, D, P, fmt)
    T = sum(news)
    g = torch.Generator().manual_seed(seed + 2)
    k, v, q = ((torch.randn((T, n, D), generator=g) * x_scale).to(dtype) for n in (H, H, H * G))
    w = [(1 + 0.3 * torch.randn((D,), generator=g)) if norm else None for _ in range(2)]
    inv = None if rot is None else (1e6 ** (-torch.arange(0, rot or D, 2, dtype=torch.float64) / (rot or D))).float()
    starts = [sum(news[:s]) for s in range(len(news) + 1)]
    batch = KVBatch(table.to(cuda), i32(lengths, cuda),
                    q_start=None if news == [1] * len(news) else i32(starts, cuda))
    dev = [None if x is None else x.to(cuda) for x in (k, v, q, w[0], w[1], inv, positions)]
    out = q4rdna.kv_append(cache, batch, dev[0], dev[1], q=dev[2], q_norm=dev[3], k_norm=dev[4], inv_freq=dev[5],
                           rotary_dim=rot or 0, rope=q4rdna.ROPE_NEOX if neox else q4rdna.ROPE_NORM,
                           positions=dev[6], q_out=dev[2] if in_place else None)
    assert q4rdna.take_fault() == 0
    pos = positions if positions is not None else torch.cat(
        [torch.arange(n) + L - n for n, L in zip(news, lengths)] or [torch.zeros(0)])
    y, mag = ref.turned(q, w[0], pos, inv, rot, neox, 1e-6)
    bound = 32 * ref.U * mag + ref.HALF[dtype] * (y.abs() + 32 * ref.U * mag) + 1e-30
    assert out.dtype == dtype and ((out.double().cpu() - y).abs() <= bound).all()
    kk, _ = ref.turned(k, w[1], pos, inv, rot, neox, 1e-6)
    ref.check_append(tiles, cache.tiles.cpu(), D, fmt, table, lengths, news, kk, v.double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt", [KV_INT8, KV_E4M3])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_append(cuda, D, fmt, dtype):
    run_append(cuda, 900 + D, [1, 16, 17, 40, 33, 600], [1, 16, 17, 9, 3, 70], 2, 4, D, 32, fmt, dtype, rot=0)
    run_append(cuda, 910 + D, [1, 2, 16, 17, 32, 100], [1] * 6, 3, 2, D, 16, fmt, dtype, rot=0)


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("rot,norm", [(None, False), (None, True), (0, False), (16, True), (32, True), (48, False)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_append_rotations(cuda, D, rot, norm, neox):
    run_append(cuda, 920 + D, [50, 21], [20, 1], 2, 3, D, 16, KV_INT8, torch.float32, neox, rot, norm)


def test_append_positions(cuda):
    """Far positions (f64 angles), positions of their own, and none of the tokens' own."""
    run_append(cuda, 930, [20, 9], [20, 4], 1, 2, 128, 16, KV_INT8, torch.float32, rot=0,
               positions=torch.randint(0, 4_000_000, (24,), generator=torch.Generator().manual_seed(3)).int())
    run_append(cuda, 931, [20, 9], [20, 4], 1, 2, 128, 16, KV_E4M3, torch.bfloat16, rot=0, neox=False,
               positions=torch.full((24,), -5).int())


def test_append_values_large_and_small(cuda):
    for scale in (1e-20, 1e-4, 1e4, 1e20):
        run_append(cuda, 940, [40, 3], [30, 2], 2, 1, 64, 16, KV_INT8, torch.float32, norm=False, x_scale=scale)
        run_append(cuda, 941, [40, 3], [30, 2], 2, 1, 64, 16, KV_E4M3, torch.float32, norm=False, x_scale=scale)


@pytest.mark.parametrize("P,H,G", [(16, 1, 1), (256, 5, 3), (64, 8, 8), (128, 1, 16)])
def test_append_layouts(cuda, P, H, G):
    run_append(cuda, 950 + P, [300, 7, 64, 257], [280, 7, 1, 2], H, G, 128, P, KV_INT8, torch.bfloat16, rot=0,
               in_place=True)


def test_append_padded_rows(cuda):
    """Rows without a token (lengths below the rows) store nothing; their q is turned all the same."""
    run_append(cuda, 960, [0, 3, 20, 0], [2, 5, 20, 40], 2, 2, 128, 16, KV_INT8, torch.float32, rot=0)
    run_append(cuda, 961, [0, 3, 0], [1, 1, 1], 2, 2, 128, 16, KV_INT8, torch.float32, rot=0)


def test_append_no_query_strided_rows(cuda):
    """Keys and values as parts of fused rows, no q, rows outside every sequence unread."""
    H, D, P = 2, 128, 16
    cache, tiles, table = make(cuda, 970, [30, 12], H, D, P, KV_INT8)
    rows = torch.randn((20, 3 * H * D))
    dev = rows.to(cuda)
    batch = KVBatch(table.to(cuda), i32([30, 12], cuda), q_start=i32([4, 9, 16], cuda))
    k, v = dev[:, : H * D], dev[:, 2 * H * D:]
    assert q4rdna.kv_append(cache, batch, k, v) is None
    part = rows[4:16].double()
    ref.check_append(tiles, cache.tiles.cpu(), D, KV_INT8, table, [30, 12], [5, 7],
                     part[:, : H * D].unflatten(1, (H, D)), part[:, 2 * H * D:].unflatten(1, (H, D)))


def test_append_not_finite(cuda):
    """A NaN or infinity makes its tile's scale NaN until the tile is begun anew; other heads and tiles are as without it."""
    H, D, P = 2, 64, 16
    cache, tiles, table = make(cuda, 980, [40], H, D, P, KV_INT8)
    for bad in (math.nan, math.inf, -math.inf):
        a, b = (KVCache(tiles.shape[0], P, H, D, tiles=tiles.to(cuda)) for _ in range(2))
        k, v = (torch.randn((20, H, D), device=cuda) for _ in range(2))
        batch = KVBatch(table.to(cuda), i32([40], cuda), q_start=i32([0, 20], cuda))
        q4rdna.kv_append(a, batch, k, v)
        k2 = k.clone()
        k2[3, 1, 7] = bad  # token 23: the second tile
        q4rdna.kv_append(b, batch, k2, v)
        sa, sb = (ref.parts(c.tiles, D, KV_INT8)[0] for c in (a, b))
        page = int(table[0, 1])
        assert torch.isnan(sb[page, 1, 0, 0]) and not torch.isnan(sa).any()
        diff = (a.tiles != b.tiles).flatten(2).any(2)
        assert diff.nonzero().tolist() == [[page, 1]]
        one = KVBatch(table.to(cuda), i32([31], cuda))
        q4rdna.kv_append(b, one, k[:1], v[:1])
        assert torch.isnan(sb[page, 1, 0, 0])  # it stays
        q4rdna.kv_append(b, KVBatch(table.to(cuda), i32([40], cuda), q_start=i32([0, 24], cuda)),
                         torch.randn((24, H, D), device=cuda), torch.randn((24, H, D), device=cuda))
        assert not torch.isnan(sb).any()


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("fmt,D", [(KV_INT8, 64), (KV_E4M3, 64), (KV_E4M3, 128), (KV_E4M3, 256)])
def test_append_not_finite_spoils_only_rows_that_see_it(cuda, fmt, D, bad, which):
    """A NaN or infinity is appended, then attended over: rows behind it in the causal order, or with a window that has
    passed its tile, are as without it; rows that see the tile are NaN.  Few and many columns, with and without a window."""
    H, G, P, L, at = 2, 4, 16, 300, 70  # token 70: tile 64..79
    clean, tiles, table = make(cuda, 985, [L], H, D, P, fmt)
    dirty = KVCache(tiles.shape[0], P, H, D, format=fmt, tiles=tiles.to(cuda))
    g = torch.Generator().manual_seed(9)
    rows = {n: torch.randn((L, H, D), generator=g).to(cuda) for n in "kv"}
    whole = KVBatch(table.to(cuda), i32([L], cuda), q_start=i32([0, L], cuda))
    q4rdna.kv_append(clean, whole, rows["k"], rows["v"])
    rows[which] = rows[which].clone()
    rows[which][at, 1, 5] = bad
    q4rdna.kv_append(dirty, whole, rows["k"], rows["v"])
    for n in (1, 3, 40, 280):
        for last in (L, 100, 82, 66):
            if n > last:
                continue
            batch = KVBatch(table.to(cuda), i32([last], cuda), q_start=i32([0, n], cuda))
            q = torch.randn((n, H * G, D), generator=g).to(cuda)
            for dtype in (torch.float32, torch.bfloat16):
                for window in (0, 10):
                    a, b = (q4rdna.kv_attention(c, batch, q.to(dtype), window=window) for c in (clean, dirty))
                    tok = torch.arange(last - n, last, device=cuda)
                    sees = (tok >= 64) & ((tok - (window or L + 1) + 1) <= 79)
                    hit = torch.zeros((n, H * G), dtype=torch.bool, device=cuda)
                    hit[:, G:] = sees[:, None]
                    assert torch.equal(b[~hit], a[~hit]) and torch.isfinite(a).all(), (n, last, dtype, window)
                    assert torch.isnan(b[hit]).all(), (n, last, dtype, window)
    # one token more in the spoilt tile, and the tile begun anew
    batch = KVBatch(table.to(cuda), i32([72], cuda))
    q4rdna.kv_append(dirty, batch, rows["k"][:1], rows["v"][:1])
    for c in ref.parts(dirty.tiles, D, fmt)[1:]:
        assert torch.isfinite(c.float()).all()


def test_append_tiny_values(cuda):
    """Values whose scale would fall under 2^-100 are stored as zeros, scale 0."""
    H, D = 1, 64
    cache = KVCache(2, 16, H, D, tiles=torch.full((2, 1, 1, 16 + 32 * D), 0xFF, dtype=torch.uint8, device=cuda))
    batch = KVBatch(i32([[1]], cuda), i32([3], cuda), q_start=i32([0, 3], cuda))
    x = torch.full((3, H, D), 1e-35, device=cuda)
    q4rdna.kv_append(cache, batch, x, torch.zeros_like(x))
    s, k, v = ref.parts(cache.tiles, D, KV_INT8)
    assert not s[1].any() and not k[1, :, :, :3].any() and not v[1, :, :, :3].any()
    assert (cache.tiles[0] == 0xFF).all()


def test_token_by_token_equals_the_definition(cuda):
    """33 single appends, each checked on the one before: scales grow, older codes follow."""
    H, D, P = 2, 128, 16
    for fmt in (KV_INT8, KV_E4M3):
        cache, tiles, table = make(cuda, 990, [33], H, D, P, fmt)
        g = torch.Generator().manual_seed(4)
        before = tiles
        for n in range(1, 34):
            k, v = (torch.randn((1, H, D), generator=g) * (1 + n % 7) for _ in range(2))
            q4rdna.kv_append(cache, KVBatch(table.to(cuda), i32([n], cuda)), k.to(cuda), v.to(cuda))
            after = cache.tiles.cpu()
            ref.check_append(before, after, D, fmt, table, [n], [1], k.double(), v.double(), f"token {n}")
            before = after


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt", [KV_INT8, KV_E4M3])
@pytest.mark.parametrize("D,P", [(64, 16), (128, 64), (256, 32)])
def test_dequant(cuda, D, P, fmt, dtype):
    cache, tiles, _ = make(cuda, 1000, [3 * P], 3, D, P, fmt)
    pages = [2, 0, 2, 4]
    k, v = q4rdna.kv_dequant(cache, i32(pages, cuda), dtype=dtype)
    s, kc, vc = ref.parts(tiles, D, fmt)
    for got, i, c in ((k, 0, kc), (v, 1, vc)):
        want = (c.float() * s[..., i, None, None]).flatten(2, 3)[pages].to(dtype)
        assert torch.equal(got.cpu(), want)


# ------------------------------------------------- streams, graphs, the chain

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_attention_between_products_of_16_columns(cuda, dtype):
    """Kernels with tensor memory of their own on both sides, each one set up while the one before it ends."""
    H, G, D, n = 2, 8, 64, 16
    cache, tiles, table = make(cuda, 1150, [900], H, D, 32, KV_INT8)
    batch = KVBatch(table.to(cuda), i32([900], cuda), q_start=i32([0, n], cuda))
    w = torch.from_numpy(synth.tiles_np(H * G * D, 512, 9)).to(cuda)
    x = torch.randn((n, 512), device=cuda)
    y, z = torch.zeros((n, H * G * D), device=cuda), torch.zeros((n, H * G * D), device=cuda)
    first, last = q4rdna.Plan([{"tiles": w, "x": x, "y": y}], B=n), q4rdna.Plan([{"tiles": w, "x": x, "y": z}], B=n)
    rows = torch.randn((n, H * G, D), device=cuda).to(dtype)

    def chain():
        for _ in range(20):
            first.run()
            out = q4rdna.kv_attention(cache, batch, rows)
            last.run()
        return out

    chain()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = chain()
    for _ in range(5):
        g.replay()
    torch.cuda.synchronize()
    assert q4rdna.take_fault() == 0 and torch.equal(y, z)
    ref.check_attention(out, ref.attention(tiles, D, KV_INT8, table, [900], [n], rows.cpu()), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fmt", [KV_INT8, KV_E4M3])
@pytest.mark.parametrize("n", [1, 24])
def test_attention_directly_behind_appends(cuda, n, fmt, dtype):
    """Steps of one token (and of 24: the kernel for many columns) over pages of 16, nothing awaited between append
    and attention: the step that fills a tile's slot 15, whose bytes share a sector with the next head's scales,
    and the one that begins the next tile are checked on the cache as it stood."""
    H, G, D, P, steps = 8, 4, 128, 16, 49 if n == 1 else 8
    cache, _, table = make(cuda, 1160, [n * steps] * 2, H, D, P, fmt)
    g = torch.Generator().manual_seed(7)
    dev = table.to(cuda)
    start = i32([0, n, 2 * n], cuda)
    rows = [[torch.randn((2 * n, h, D), generator=g).to(dtype).to(cuda) for h in (H, H, H * G)] for _ in range(steps)]
    batches = [KVBatch(dev, i32([n * i, n * i], cuda), q_start=start) for i in range(1, steps + 1)]
    kept = []
    torch.cuda.synchronize()
    for i, ((k, v, q), batch) in enumerate(zip(rows, batches), 1):
        q4rdna.kv_append(cache, batch, k, v)
        out = q4rdna.kv_attention(cache, batch, q)
        if n > 1 or i % 16 < 2:
            kept.append((i, q, out, cache.tiles.clone()))
    for i, q, out, tiles in kept:
        want = ref.attention(tiles.cpu(), D, fmt, table, [n * i] * 2, [n, n], q.cpu())
        ref.check_attention(out, want, dtype, f"step {i}")
    assert q4rdna.take_fault() == 0


def test_side_stream_and_graphs(cuda):
    """Two captured calls replayed on two streams at once, lengths changed between
    replays; and a call on a stream that is not current."""
    H, G, D, P = 2, 4, 128, 16
    lengths = [3000, 40]
    cache, tiles, table = make(cuda, 1100, lengths, H, D, P, KV_INT8)
    dev_len = i32(lengths, cuda)
    one = KVBatch(table.to(cuda), dev_len)
    few = KVBatch(table.to(cuda), dev_len, q_start=i32([0, 40, 50], cuda))
    q1, q2 = torch.randn((2, H * G, D), device=cuda), torch.randn((50, H * G, D), device=cuda)
    q3 = q2.bfloat16()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    a = q4rdna.kv_attention(cache, one, q1, stream=side)
    b = q4rdna.kv_attention(cache, one, q1)
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    graphs, outs = [], []
    for batch, q in ((one, q1), (few, q2), (few, q3)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(q4rdna.kv_attention(cache, batch, q))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for lengths in ([3000, 40], [1000, 33], [41, 11]):
        dev_len.copy_(i32(lengths, cuda))
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        ref.check_attention(outs[0], ref.attention(tiles, D, KV_INT8, table, lengths, [1, 1], q1.cpu()), torch.float32)
        for o, q in ((outs[1], q2), (outs[2], q3)):
            ref.check_attention(o, ref.attention(tiles, D, KV_INT8, table, lengths, [40, 10], q.cpu()), q.dtype)
    assert q4rdna.take_fault() == 0


def test_attention_is_deterministic(cuda):
    cache, _, table = make(cuda, 1200, [5000, 900, 77], 2, 128, 32, KV_E4M3)
    for news, dtype in (([1, 1, 1], torch.float32), ([4, 1, 2], torch.float32), ([200, 77, 1], torch.bfloat16)):
        q = torch.randn((sum(news), 8, 128), device=cuda).to(dtype)
        start = i32([0, news[0], news[0] + news[1], sum(news)], cuda)
        batch = KVBatch(table.to(cuda), i32([5000, 900, 77], cuda), q_start=start)
        first = q4rdna.kv_attention(cache, batch, q)
        for _ in range(20):
            assert torch.equal(q4rdna.kv_attention(cache, batch, q), first)


def test_workspace_is_checked(cuda):
    import ctypes

    cache, _, table = make(cuda, 1210, [5000], 2, 128, 32, KV_INT8)
    batch = KVBatch(table.to(cuda), i32([5000], cuda))
    q = torch.randn((1, 8, 128), device=cuda)
    a = q4rdna.KVAttentionArgs(0, 1, 8, q.data_ptr(), q.data_ptr(), 1024, 1024, 0.0, 0)
    batch._rec.desc.max_length = 5024
    L, ref_a, b, c = q4rdna.lib, ctypes.byref(a), ctypes.byref(batch._rec.desc), ctypes.byref(cache._rec.desc)
    n = L.q4rdna_kv_attention_workspace_bytes(c, b, ref_a)
    assert n > 0
    ws = torch.empty(n + 16, dtype=torch.uint8, device=cuda)
    assert L.q4rdna_kv_attention(c, b, ref_a, None, 0, None) == 4
    assert L.q4rdna_kv_attention(c, b, ref_a, ws.data_ptr(), n - 1, None) == 4
    assert L.q4rdna_kv_attention(c, b, ref_a, ws.data_ptr() + 8, n, None) == 3


@pytest.mark.parametrize("tokens", [1, 5])
def test_decoder_attention_block(cuda, tokens):
    """The block as a decoder runs it: RMSNorm + q/k/v products (one plan), append
    with per-head norm and rotation, attention, output product + residual; steps
    of 1 and 5 tokens on one sequence, the attention checked on the cache as it
    then stands and the products on the attention's outputs."""
    hid, H, G, D, P = 512, 2, 4, 64, 16
    Hq = H * G
    shapes = {"q": (Hq * D, hid), "k": (H * D, hid), "v": (H * D, hid), "o": (hid, Hq * D)}
    tiles = {n: torch.from_numpy(synth.tiles_np(N, K, 20 + i)).to(cuda) for i, (n, (N, K)) in enumerate(shapes.items())}
    W = {n: q4rdna.dequant(t, *shapes[n]).double().cpu() for n, t in tiles.items()}
    g = torch.Generator().manual_seed(6)
    gn, qn, kn = ((1 + 0.1 * torch.randn((n,), generator=g)).to(cuda) for n in (hid, D, D))
    inv = (1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().to(cuda)
    cache = KVCache(8, P, H, D)
    table = torch.tensor([[5, 0, 7, 2]], dtype=torch.int32)
    h = torch.zeros((tokens, hid), device=cuda)
    y = {n: torch.zeros((tokens, shapes[n][0]), device=cuda) for n in "qkv"}
    plan = q4rdna.Plan([{"tiles": tiles[n], "x": h, "y": y[n], "norm_weight": gn} for n in "qkv"], B=tokens)
    lengths = i32([0], cuda)
    batch = KVBatch(table.to(cuda), lengths, q_start=i32([0, tokens], cuda))
    for step in range(1, 60 // tokens):
        h.copy_(torch.randn((tokens, hid), generator=g))
        lengths.fill_(step * tokens)
        before = cache.tiles.cpu()
        plan.run()
        q = q4rdna.kv_append(cache, batch, y["k"], y["v"], q=y["q"], inv_freq=inv, q_norm=qn, k_norm=kn)
        att = q4rdna.kv_attention(cache, batch, q)
        out = q4rdna.gemv(tiles["o"], att, op=q4rdna.OP_ADD, add=h)
        if step % 4 != 1:
            continue
        x = h.double().cpu()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gn.double().cpu()
        got = {n: y[n].double().cpu() for n in "qkv"}
        for n in "qkv":  # the products' own tolerance (tests/tolerance.py)
            assert ((got[n] - x @ W[n].T).abs() <= 1e-5 * (x.abs() @ W[n].abs().T)).all()
        pos = torch.arange(step * tokens - tokens, step * tokens)
        L = [step * tokens]
        kk, _ = ref.turned(got["k"].unflatten(1, (H, D)), kn.cpu(), pos, inv.cpu(), 0, True, 1e-6)
        tiles_now = cache.tiles.cpu()
        ref.check_append(before, tiles_now, D, KV_INT8, table, L, [tokens], kk, got["v"].unflatten(1, (H, D)))
        qq, mag = ref.turned(got["q"].unflatten(1, (Hq, D)), qn.cpu(), pos, inv.cpu(), 0, True, 1e-6)
        qd = q.unflatten(1, (Hq, D)).double().cpu()
        assert ((qd - qq).abs() <= 32 * ref.U * mag + ref.U * qq.abs()).all()
        want = ref.attention(tiles_now, D, KV_INT8, table, L, [tokens], q.cpu().unflatten(1, (Hq, D)))
        ref.check_attention(att.unflatten(1, (Hq, D)), want, torch.float32)
        a = att.double().cpu()
        o = a @ W["o"].T + h.double().cpu()
        assert ((out.double().cpu() - o).abs() <= 1e-5 * (a.abs() @ W["o"].abs().T + h.abs().cpu())).all()
    assert q4rdna.take_fault() == 0


@pytest.mark.parametrize("model,batch", [("qwen3-8b", 1), ("qwen3-32b", 9)])
def test_bench_runs_a_decoder_step(cuda, model, batch):
    """bench.py --attention: one layer, a cache whose last page is not full."""
    import json
    import os
    import subprocess
    import sys

    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(repo, "bench.py"), "--attention", "203", "--layers", "1", "--model",
                        model, "--batch", str(batch), "--steps", "3", "--warmup", "3"], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    out = json.loads(r.stdout)
    assert out["config"]["kv_heads"] == 8 and out["config"]["heads"] == (32 if model == "qwen3-8b" else 64)
    assert out["gpu_launches"] > 0 and 0 < out["append_attention_us"] < out["value"] < 1e5
