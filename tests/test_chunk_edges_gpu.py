"""Chunk operators where their numbers are hard: int8 value rows of zeros and
of scales far apart, infinities and NaN, rows whose first keys count for
nothing, caches without a block to spare. Every result has to be finite where
the definition's is, and within the bound; the definition is computed in 64
bits from the codes and scales that the cache holds.

Tolerances. Half a step is 2^-8 of a bf16 value, 2^-11 of an f16, 2^-24 of an
f32. A softmax weight is off by
  - its rounding: bf16 caches 2^-8; int8 caches, whose weights times the value's
    scale s are f16 in a unit in which the row's largest p s is 2^6 at least,
    2^-11, or 2^-25 / 2^6 of that largest below f16's least normal number,
  - its score, a sum of D products in f32: 2 D 2^-24 B, B the largest
    scale * sum |q k| that the row sees,
  - the exponent, score + log2 s less the row's reference: at most eight
    roundings of numbers up to 2 (B log2 e + max |log2 s| + 14):
    2^-20 (B log2 e + max |log2 s| + 14),
  - the exponential and the sums: 2^-20.
E is the sum of the last three, w the rounding. With A = sum of p |v|:
  |out - exact| <= 2^-8 |exact| + (1 + 2^-8) ((w + E) A + n 127 max(p s) 2^-31)
  |lse - exact| <= E + 2^-22 |exact|
and 127 * 2^-100 for V scales under 2^-100, which count as that.
"""
import math

import numpy as np
import pytest

from tests.test_chunk_ops_gpu import CHUNKS, FEW, KV, RUNS, SM, make, rnd  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def held(c, layer, s):
    """(k, v, V scales) of a sequence in 64 bits: [len, H, D] twice and [len, H] (0 for rows of zeros; None in bf16)."""
    n, bs = c.seq_len(layer, s), c.block_size
    p, t = c.pages(), torch.arange(n, device="cuda")
    blocks = torch.tensor(c.block_table(layer, s), dtype=torch.long, device="cuda")[t // bs] if n else t
    k, v = (p[x][blocks, :, t % bs].double() for x in ("k", "v"))
    if "k_scale" not in p:
        return k, v, None
    sk, sv = (p[x + "_scale"][blocks, :, t % bs].double() for x in ("k", "v"))
    return k * sk[..., None], v * sv[..., None], torch.where((v == 0).all(-1), 0.0, sv)


def definition(q, k, v, sv, m, causal):
    """out, lse and their tolerances; what a row does not see never enters."""
    n, hkv, D = k.shape
    G, scale = q.shape[1] // hkv, 1 / math.sqrt(D)
    k, v = (t.repeat_interleave(G, 1) for t in (k, v))
    q = q.double()
    last = torch.arange(m, device=q.device) + (n - m) if causal else torch.full((m,), n - 1, device=q.device)
    sees = (torch.arange(n, device=q.device)[None] <= last[:, None])[:, None]
    s = (torch.einsum("mhd,nhd->mhn", q, k) * scale).masked_fill(~sees, -math.inf)
    if n == 0:
        none = torch.full((m, q.shape[1]), -math.inf, device=q.device, dtype=torch.float64)
        zero = torch.zeros(m, q.shape[1], D, device=q.device, dtype=torch.float64)
        return zero, none, zero, torch.zeros_like(none)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None]).nan_to_num(0.0)
    hide = (p == 0)[..., None] & ~torch.isfinite(v).transpose(0, 1)[None] if not bool(torch.isfinite(v).all()) else None
    if hide is None:
        out, a = torch.einsum("mhn,nhd->mhd", p, v), torch.einsum("mhn,nhd->mhd", p, v.abs())
    else:
        pv = (p[..., None] * v.transpose(0, 1)[None]).masked_fill(hide, 0.0)
        out, a = pv.sum(2), pv.abs().sum(2)
    b = (torch.einsum("mhd,nhd->mhn", q.abs(), k.abs()) * scale).masked_fill(~sees | torch.isinf(s), 0.0).amax(-1)
    tiny = torch.zeros_like(b)
    mag = b * math.log2(math.e) + 14
    if sv is not None:
        sv = sv.repeat_interleave(G, 1)
        ok = torch.isfinite(sv) & (sv > 0)
        spread = torch.where(ok, sv, 1.0).log2().abs().amax(0)
        mag = mag + spread
        tiny = 127 * (n * 2.0 ** -31 * (p * torch.where(ok, sv, 0.0).transpose(0, 1)).amax(-1) + 2.0 ** -100)
    e = 2 * D * 2.0 ** -24 * b + 2.0 ** -20 * mag + 2.0 ** -20
    w = 2.0 ** -8 if sv is None else 2.0 ** -11
    tol = 2.0 ** -8 * out.abs() + (1 + 2.0 ** -8) * ((w + e[..., None]) * a + tiny[..., None]) + 2.0 ** -130
    return out, lse, tol, e + 2.0 ** -22 * lse.abs()


def check(out, lse, q, c, layer, ids, counts, causal=True, rows=None, lse_only=False):
    """Every row (or those of `rows`, a mask over the packed ones) against the definition."""
    at = 0
    for s, m in zip(ids, counts):
        o, z, to, tz = definition(q[at:at + m], *held(c, layer, s), m, causal)
        g, y = out[at:at + m].double(), lse[at:at + m].double()
        if rows is not None:
            o, z, to, tz, g, y = (t[rows[at:at + m]] for t in (o, z, to, tz, g, y))
        none = torch.isinf(z)
        assert torch.equal(torch.isinf(y) & (y < 0), none), s
        dz = (y - z)[~none].abs()
        assert bool((dz <= tz[~none]).all()), (s, "lse", float(dz.max()), float(tz[~none].max()))
        if not lse_only:
            assert bool(torch.isfinite(to).all()) and bool((g[none] == 0).all()), s
            off = (g - o).abs()
            assert bool((off <= to).all()), (s, float((off / to).nan_to_num(math.inf).max()), int((~(off <= to)).sum()))
        at += m


def attend(c, ids, counts, q, causal=True, **kw):
    lse = torch.full((q.shape[0], q.shape[1]), 7.0, device="cuda")
    out = c.chunk_attention(0, ids, counts, q, causal=causal, lse=lse)
    check(out, lse, q, c, 0, ids, counts, causal, **kw)
    return out, lse


def filled(KV, k, v, int8, bs=16):
    n, H, D = k.shape
    c = make(KV, 1, H, D, bs, -(-n // bs) + 2, 1, int8)
    c.append_chunks(0, [0], [n], k, v)
    return c


ROWS = [150, 60, 24, 5]  # queries of a chunk: the many-row kernel, and the few-row one with 64, 32 and 16 columns
SHAPES = [(2, 600), (2, 1500), (16, 1500)]  # heads, keys: whole items, items cut tile by tile, items cut into pieces of several


# ---------------------------------------------------------------- attention over int8 caches

@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("big,small", [(2.0 ** 115, 2.0 ** -20), (2.0 ** 120, 1.0), (2.0 ** 100, 2.0 ** -90), (2.0 ** 30, 2.0 ** -30)])
@pytest.mark.parametrize("where", ["first", "last", "each tile", "one"])
def test_int8_equal_scores_and_value_scales_far_apart(KV, D, m, big, small, where):
    # the sum of the weights knows nothing of the values' sizes
    for H, n in SHAPES:
        k, v = torch.zeros(n, H, D, dtype=torch.bfloat16, device="cuda"), rnd((n, H, D), 2, small)
        at = {"first": slice(0, 200), "last": slice(400, n), "each tile": slice(7, n, 50), "one": slice(3, 4)}[where]
        v[at] = rnd((n, H, D), 3, big)[at]
        attend(filled(KV, k, v, True), [0], [m], rnd((m, H, D), 4))


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size,logit", [(1.0, 0.0), (0.02, 10.0), (0.002, 12.0), (1e-4, 12.0), (1e-4, 30.0), (1.0, 100.0)])
@pytest.mark.parametrize("where", ["one", "some", "first", "all"])
def test_int8_value_rows_of_zeros(KV, D, m, size, logit, where):
    # padding or an attention sink: nothing for the output, a share of the sum
    for H, n in SHAPES:
        k, v, q = rnd((n, H, D), 1), rnd((n, H, D), 2, size), rnd((m, H, D), 3)
        at = {"one": slice(5, 6), "some": slice(3, n, 41), "first": slice(0, 300), "all": slice(0, n)}[where]
        q[..., 0], k[..., 0] = 4.0, 0.0
        k[at, :, 0] = logit * math.sqrt(D) / 4.0
        v[at] = 0.0
        attend(filled(KV, k, v, True), [0], [m], q)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [3, 5, 7, 48])
def test_int8_unusual_scales_beside_rows_without_a_token(KV, G, D, causal):
    # 128 is no multiple of G: a tile's last rows hold no token, but what an
    # earlier call left in shared memory, here values that make scores infinite
    H, lens, counts = 1, [319, 8, 83, 530, 118, 700], [319, 8, 64, 17, 65, 2]
    for far in (True, False):
        k, v, q = rnd((sum(lens), H, D), 1), rnd((sum(lens), H, D), 2), rnd((sum(counts), H * G, D), 3)
        v[3::11] *= 2.0 ** 60 if far else 0.0
        c = make(KV, 1, H, D, 16, sum(-(-x // 16) for x in lens), len(lens), True)
        c.append_chunks(0, range(len(lens)), lens, k, v)
        first = attend(c, range(len(lens)), counts, q, causal)
        for scale in (3e38, 1e4, 0.0):
            c.chunk_attention(0, range(len(lens)), counts, torch.full_like(q, scale) * k.new_tensor([1.0, -1.0]).repeat(D // 2), causal=causal)
            for a, b in zip(first, attend(c, range(len(lens)), counts, q, causal)):
                assert torch.equal(a, b), "not deterministic"


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("D", [64, 128])
def test_int8_rows_of_full_range_are_not_zeros(KV, D, m):
    # scale 1 as a row of zeros has, but with codes; the first values are 0
    H, n = 2, 400
    k, v = rnd((n, H, D), 1), torch.zeros(n, H, D, dtype=torch.bfloat16, device="cuda")
    v[..., D - 1], v[::2, :, D - 2] = 127.0, -127.0
    v[::3] = rnd((n, H, D), 2, 1e-3)[::3]
    attend(filled(KV, k, v, True), [0], [m], rnd((m, H, D), 3))


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("m", [200, 64, 20])
@pytest.mark.parametrize("D", [64, 128])
def test_int8_values_that_are_not_finite(KV, D, m, bad):
    # a value row with an infinity has the scale inf: NaN for the rows that see
    # it, whose lse knows nothing of it; nothing for the others
    H, n, at = 2, 300, 290
    k, v, q = rnd((n, H, D), 1), rnd((n, H, D), 2), rnd((m, H, D), 3)
    if math.isinf(bad):
        v[at, 0, 3] = bad
    c = filled(KV, k, v, True)
    if math.isnan(bad):
        c.pages()["v_scale"][c.block_table(0, 0)[at // 16], 0, at % 16] = bad
    lse = torch.full((m, H), 7.0, device="cuda")
    out = c.chunk_attention(0, [0], [m], q, lse=lse)
    sees = torch.arange(m, device="cuda") + n - m >= at
    check(out, lse, q, c, 0, [0], [m], lse_only=True)
    check(out, lse, q, c, 0, [0], [m], rows=~sees)
    assert bool(torch.isnan(out[sees, 0]).all()) and bool(torch.isfinite(out[:, 1]).all())


# ---------------------------------------------------------------- attention, both caches

@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("score", [-3.0, -60.0, -150.0, 150.0])
def test_keys_of_score_minus_infinity_before_the_others(KV, D, m, score):
    # a row's unit comes from the first key that counts, not from the first key
    for H, n in SHAPES:
        k, v, q = rnd((n, H, D), 1), rnd((n, H, D), 2), rnd((m, H, D), 3)
        q[..., 0], q[..., 1] = 1.0, 8.0
        k[..., 0], k[..., 1] = 0.0, score * math.sqrt(D) / 8.0
        k[:260, :, 0] = -math.inf
        attend(filled(KV, k, v, False), [0], [m], q)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H,G,D,bs,lens,counts", CHUNKS + [(x[0], x[1], D, *x[2:]) for x in FEW + RUNS for D in (64, 128)])
def test_every_row_is_finite_and_within_the_bound(KV, H, G, D, bs, lens, counts, int8):
    n = len(lens)
    c = make(KV, 1, H, D, bs, sum(-(-x // bs) for x in lens), n, int8)
    v = rnd((sum(lens), H, D), 2)
    v[::5] *= 100.0
    v[1::7] *= 0.001
    c.append_chunks(0, range(n), lens, rnd((sum(lens), H, D), 1), v)
    for causal in (True, False):
        attend(c, range(n), counts, rnd((sum(counts), H * G, D), 3, 2.0), causal)


@pytest.mark.parametrize("int8", [False, True])
def test_rows_that_see_nothing_and_rows_that_do(KV, int8):
    H, D = 2, 128
    c = make(KV, 1, H, D, 16, 32, 8, int8)
    c.append_chunks(0, [1, 2, 3], [3, 150, 16], rnd((169, H, D), 1), rnd((169, H, D), 2))
    c.truncate([3], [0])
    ids, counts = [1, 4, 3, 2, 1], [9, 5, 2, 140, 0]
    for causal in (True, False):
        attend(c, ids, counts, rnd((sum(counts), 4, D), 3), causal)


@pytest.mark.parametrize("int8", [False, True])
def test_attention_behind_four_gigabytes_is_finite(KV, int8):
    H, D, bs = 32, 128, 1024
    fill = 1100 if int8 else 560
    c = make(KV, 1, H, D, bs, fill + 4, fill + 1, int8)
    one = rnd((fill, H, D), 0)
    c.append_chunks(0, range(fill), [1] * fill, one, one)
    n = 2500
    v = rnd((n, H, D), 2)
    v[9::100] = 0.0
    c.append_chunks(0, [fill], [n], rnd((n, H, D), 1), v)
    assert min(c.block_table(0, fill)) * H * bs * D * (1 if int8 else 2) > 2 ** 32
    for m in (3, 70):
        attend(c, [fill], [m], rnd((m, H, D), 3, 2.0))


def test_chunk_attention_refuses_what_is_no_tensor_and_scales_that_overflow(KV):
    from vortex_b200 import _native as N
    c = filled(KV, rnd((20, 2, 64), 1), rnd((20, 2, 64), 2), False)
    q = rnd((4, 2, 64), 3)
    for args in (dict(q=q.cpu().float().numpy()), dict(q=None), dict(lse=[[0.0, 0.0]] * 4), dict(lse=q.float().cpu().numpy()[..., 0]),
                 dict(softmax_scale=3e38), dict(softmax_scale=1e39)):
        with pytest.raises(N.VxbError) as e:
            c.chunk_attention(0, [0], [4], **{"q": q, **args})
        assert e.value.code == N.VXB_EINVAL
    out = c.chunk_attention(0, [0], [4], torch.zeros_like(q), softmax_scale=2e38)
    assert bool(torch.isfinite(out).all())


# ---------------------------------------------------------------- cache

def test_truncate_of_every_holder_needs_the_blocks_it_frees(KV):
    # a full pool; both holders of every block are cut: two blocks come free
    # and one copy of the block with the cut is needed
    k = rnd((64, 1, 64), 0)
    c = make(KV, 1, 1, 64, 16, 4, 2)
    c.append_chunks(0, [0], [64], k, -k)
    c.fork(0, 1, 64)
    assert c.free_block_count() == 0
    c.truncate([0, 1], [20, 20])
    assert c.free_block_count() == 1 and c.block_table(0, 0)[0] == c.block_table(0, 1)[0]
    assert c.block_table(0, 0)[1] != c.block_table(0, 1)[1]
    for s in (0, 1):
        gk, gv = c.get_kv(0, s)
        assert torch.equal(gk, k[:20].float()) and torch.equal(gv, -k[:20].float())


@pytest.mark.parametrize("blocks", [7, 6])
def test_truncate_of_several_holders_at_different_places(KV, blocks):
    # two cuts inside block 2, which the fourth sequence keeps, one inside block
    # 0, which all others keep: three copies
    from vortex_b200 import _native as N
    k = rnd((64, 1, 64), 0)
    c = make(KV, 1, 1, 64, 16, blocks, 4)
    c.append_chunks(0, [0], [64], k, -k)
    for s in (1, 2, 3):
        c.fork(0, s, 64)
    lens = [40, 47, 9, 64]
    if blocks == 6:
        with pytest.raises(N.VxbError) as e:
            c.truncate(range(4), lens)
        assert e.value.code == N.VXB_ENOBLOCKS
        lens = [64] * 4
    else:
        c.truncate(range(4), lens)
        assert c.free_block_count() == 0
        assert len({c.block_table(0, s)[2] for s in (0, 1, 3)}) == 3
    for s in range(4):
        gk, gv = c.get_kv(0, s)
        assert torch.equal(gk, k[:lens[s]].float()) and torch.equal(gv, -k[:lens[s]].float())


def test_truncate_without_a_block_to_spare_changes_nothing(KV):
    from vortex_b200 import _native as N
    k = rnd((64, 1, 64), 0)
    c = make(KV, 1, 1, 64, 16, 4, 3)
    c.append_chunks(0, [0], [64], k, -k)
    c.fork(0, 1, 64)
    before = c.stats(), [c.block_table(0, s) for s in (0, 1)], c.pages()["lens"].tolist()
    with pytest.raises(N.VxbError) as e:
        c.truncate([0], [20])  # the other sequence keeps every block
    assert e.value.code == N.VXB_ENOBLOCKS
    assert (c.stats(), [c.block_table(0, s) for s in (0, 1)], c.pages()["lens"].tolist()) == before
    # cut inside a block that stays shared with one that is cut behind it
    with pytest.raises(N.VxbError) as e:
        c.truncate([0, 1], [20, 64])
    assert e.value.code == N.VXB_ENOBLOCKS
    assert (c.stats(), [c.block_table(0, s) for s in (0, 1)], c.pages()["lens"].tolist()) == before


def test_an_append_that_cannot_be_launched_takes_nothing(KV):
    # a stream whose capture has been broken off takes no launches: the host's
    # tables and the device's lengths stay as they were, and later calls work
    import ctypes
    from vortex_b200 import _native as N
    rt = ctypes.CDLL("libcudart.so.12")
    c = make(KV, 1, 2, 64, 16, 700, 400)
    k = rnd((5000, 2, 64), 0)
    c.append_chunks(0, [1, 2], [20, 3], k[:23], k[:23])
    torch.cuda.synchronize()
    before = c.free_block_count(), [c.block_table(0, s) for s in (1, 2)], c.pages()["lens"].tolist()
    side = torch.cuda.Stream()
    raw, graph = ctypes.c_void_p(side.cuda_stream), ctypes.c_void_p()
    assert rt.cudaStreamBeginCapture(raw, 0) == 0
    assert rt.cudaStreamSynchronize(raw) != 0  # not allowed in a capture, which ends with it
    with torch.cuda.stream(side):
        for ids, counts in (([1, 2], [30, 1]), (list(range(1, 301)), [9] * 300)):
            with pytest.raises(N.VxbError) as e:
                c.append_chunks(0, ids, counts, k[:sum(counts)], k[:sum(counts)])
            assert e.value.code == N.VXB_ECUDA and "append" in str(e.value)
    assert rt.cudaStreamEndCapture(raw, ctypes.byref(graph)) != 0
    rt.cudaGetLastError()
    assert c.free_block_count() == before[0] and [c.block_table(0, s) for s in (1, 2)] == before[1] and [c.seq_len(0, s) for s in (1, 2, 3)] == [20, 3, 0]
    assert c.pages()["lens"].tolist() == before[2]
    c.append_chunks(0, [1, 2], [30, 1], k[23:54], k[23:54])
    assert torch.equal(c.get_kv(0, 1)[0], torch.cat([k[:20], k[23:53]]).float())


def test_append_int8_scales_of_keys_and_values(KV):
    D = 64
    rows = [torch.linspace(-1, 1, D) * m * (1 + j / 16) for m in (1.0, 127.0, 3.0, 1e-38, 1e38, 2.0 ** -133) for j in range(16)]
    rows += [torch.zeros(D), torch.full((D,), 5.0), torch.tensor([math.inf] + [1.0] * (D - 1)), torch.tensor([math.nan] * D)]
    k = torch.stack(rows)[:, None].to(torch.bfloat16).cuda()
    a, b = (make(KV, 1, 1, D, 16, 16, 1, True) for _ in range(2))
    a.append_chunks(0, [0], [k.shape[0]], k, -k.flip(0))
    b.append_seq(0, 0, k, -k.flip(0))
    pa, pb = a.pages(), b.pages()
    for name in ("k", "v"):
        assert torch.equal(pa[name], pb[name])
        assert torch.equal(pa[name + "_scale"].view(torch.int32), pb[name + "_scale"].view(torch.int32))


# ---------------------------------------------------------------- probabilities

@pytest.mark.parametrize("rows,vocab", [(2, 2000), (300, 30001)])
@pytest.mark.parametrize("t", [0.011, 1.4091, 0.3])
def test_probs_far_below_the_maximum(SM, rows, vocab, t):
    # d = x - max is off by 2^-24 of it, log2(e) / t and their product by 2^-24
    # each, so the exponent by 3 * 2^-24 |d| / t; the exponential by 2^-22, the
    # sums by at most 64 * 2^-24 and two more roundings: 2^-17 in all
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = -85.0 * t * torch.rand(rows, vocab, generator=g, device="cuda") + 3.0
    p = SM.token_probs(x, t).double()
    d = (x.double() - x.double().amax(-1, keepdim=True)) / t
    want = torch.softmax(d, -1)
    assert bool(((p - want).abs() <= (2.0 ** -17 + 3 * 2.0 ** -24 * d.abs()) * want + 2.0 ** -125).all())
