"""Chunk and draft operators on the GPU against plain computations in 64 bits:
ragged append, truncate, chunk attention, token probabilities, draft
verification, and a run of them together.

Tolerances. A rounding to bf16 is off by at most 2^-8 of the value, one to f32
by 2^-24. Chunk attention rounds each softmax weight (times the value's scale,
int8) to bf16 once and the output once; a score is a sum of D products in f32,
so a weight is off by 2 D 2^-24 of the sum of |q k| besides, and by 2^-20 for
the exponential and the sums of weights. With A = sum of p |v| and B the
largest scale * sum |q k| of the row:
  |out - exact| <= 2^-8 |exact| + (2^-8 + 2 D 2^-24 B + 2^-20) (1 + 2^-8) A
  |lse - exact| <= 2 D 2^-24 B + 2^-20 + 2^-22 |exact|
token_probs: d = (x - max) / t is off by 2^-23 |d|, the exponential by 2^-22,
a sum of at most 64 sequential additions by 64 * 2^-24, two more roundings:
  |p - exact| <= (2^-17 + 2^-23 |d|) exact + 2^-125.
Everything else is equal bit for bit.
"""
import math

import numpy as np
import pytest

from oracle.kv_oracle import KVOracle

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def KV(cuda_ok):
    from vortex_b200 import kv_cache
    return kv_cache


@pytest.fixture(scope="module")
def SM(cuda_ok):
    from vortex_b200 import sampling
    return sampling


def rnd(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(torch.bfloat16)


def make(KV, layers, H, D, bs, blocks, seqs, int8=False, poison=True):
    c = KV.PagedKVCache(layers, H, D, block_size=bs, max_blocks=blocks, max_seqs=seqs,
                        kv_dtype=KV.I8 if int8 else KV.BF16)
    if poison:  # what nobody wrote must never matter
        p = c.pages()
        for name in ("k", "v"):
            p[name].fill_(-128 if int8 else float("nan"))
            if int8:
                p[name + "_scale"].fill_(float("nan"))
    return c


# ---------------------------------------------------------------- append, truncate

@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H,D,bs", [(1, 64, 16), (3, 128, 16), (8, 128, 48), (2, 64, 32)])
def test_append_chunks_equals_single_appends(KV, H, D, bs, int8):
    a, b = (make(KV, 2, H, D, bs, 200, 8, int8) for _ in range(2))
    o = KVOracle(2, H, D, bs, 200)
    steps = [(0, [4, 9, 2], [5, 0, 33]), (1, [9], [17]), (0, [2, 4, 9, 7], [1, 16, 3, 47]), (1, [4, 9], [0, 31]),
             (0, [9, 2], [200, 29])]
    for step, (layer, ids, counts) in enumerate(steps):
        k, v = rnd((sum(counts), H, D), 2 * step), rnd((sum(counts), H, D), 2 * step + 1, 7.0)
        a.append_chunks(layer, ids, counts, k, v)
        at = 0
        for i, n in zip(ids, counts):
            if n:
                b.append_seq(layer, i, k[at:at + n], v[at:at + n])
            for t in range(n):
                o.append_kv(layer, i, np.zeros((H, D)), np.zeros((H, D)))
            at += n
    torch.cuda.synchronize()
    for (layer, i), table in o.tables.items():
        assert a.block_table(layer, i) == table == b.block_table(layer, i)
        assert a.seq_len(layer, i) == b.seq_len(layer, i)
    pa, pb = a.pages(), b.pages()
    for name in pa:
        x, y = pa[name], pb[name]
        x, y = (t.view(torch.int16) if t.dtype == torch.bfloat16 else t.view(torch.int32) if t.dtype == torch.float32 else t
                for t in (x, y))
        assert torch.equal(x, y), name  # what was not written is untouched too
    assert a.stats() == b.stats()


def test_append_int8_codes_on_every_rounding(KV):
    # every bf16 quotient near a half: rows v / m with m a few values, and rows
    # of zeros, of one value, of tiny and huge values, of NaN and infinities
    D = 64
    rows = []
    for m in (1.0, 127.0, 3.0, 1e-38, 1e38, 2.0 ** -133):
        for j in range(16):
            r = torch.linspace(-1, 1, D) * m * (1 + j / 16)
            rows.append(r)
    rows += [torch.zeros(D), torch.full((D,), 5.0), torch.arange(D) / 2 - 16.0, torch.arange(D) * 1.0 - 32]
    bad = torch.randn(D)
    bad[3], bad[9], bad[11] = float("nan"), float("inf"), -float("inf")
    rows.append(bad)
    k = torch.stack(rows)[:, None].to(torch.bfloat16).cuda()
    a, b = (make(KV, 1, 1, D, 16, 16, 1, True) for _ in range(2))
    a.append_chunks(0, [0], [k.shape[0]], k, -k)
    b.append_seq(0, 0, k, -k)
    pa, pb = a.pages(), b.pages()
    for name in ("k", "v"):
        assert torch.equal(pa[name], pb[name]), name
    assert torch.equal(pa["k_scale"].view(torch.int32), pb["k_scale"].view(torch.int32))


@pytest.mark.parametrize("seqs,tokens", [(150, 3), (1, 23000), (70, 301)])
def test_append_of_more_than_one_launch_holds(KV, seqs, tokens):
    H, D, bs = 1, 64, 16
    c = make(KV, 1, H, D, bs, seqs * (tokens // bs + 2), seqs)
    counts = [tokens + (i % 3) for i in range(seqs)]
    k, v = rnd((sum(counts), H, D), 1), rnd((sum(counts), H, D), 2)
    first = [1 + i % 5 for i in range(seqs)]
    c.append_chunks(0, range(seqs), first, k[:sum(first)], v[:sum(first)])
    c.append_chunks(0, range(seqs), counts, k, v)
    at = f = 0
    for i in range(seqs):
        gk, gv = c.get_kv(0, i)
        assert torch.equal(gk, torch.cat([k[f:f + first[i]], k[at:at + counts[i]]]).float())
        assert torch.equal(gv, torch.cat([v[f:f + first[i]], v[at:at + counts[i]]]).float())
        at, f = at + counts[i], f + first[i]
    assert c.pages()["lens"][0].tolist() == [a + b for a, b in zip(counts, first)]


def test_append_chunks_is_all_or_nothing(KV):
    from vortex_b200 import _native as N
    c = KV.PagedKVCache(1, 1, 64, block_size=16, max_blocks=4, max_seqs=2, max_blocks_per_seq=3)
    k = rnd((60, 1, 64), 0)
    c.append_chunks(0, [1], [20], k[:20], k[:20])
    before = c.stats()

    def refused(ids, counts, code):
        with pytest.raises(N.VxbError) as e:
            c.append_chunks(0, ids, counts, k[:sum(counts)], k[:sum(counts)])
        assert e.value.code == code
        assert c.stats() == before and c.seq_len(0, 1) == 20

    refused([2, 1], [20, 20], N.VXB_ENOBLOCKS)       # 2 + 1 blocks, 2 free
    refused([1], [29], N.VXB_ENOBLOCKS)              # a fourth block of one sequence
    refused([2, 3], [1, 1], N.VXB_ENOBLOCKS)         # a third slot
    refused([2, 2], [1, 1], N.VXB_EINVAL)
    for args in ((1, [1], [1], k[:1], k[:1]), (0, [1], [2], k[:1], k[:1]), (0, [1], [1], k[:1].float(), k[:1]),
                 (0, [1], [1], k[:1], k[:1].cpu()), (0, [1], [-1], k[:0], k[:0])):
        with pytest.raises(N.VxbError):
            c.append_chunks(*args)
    c.append_chunks(0, [1, 2], [0, 0], k[:0], k[:0])
    assert c.stats() == before
    c.append_chunks(0, [1, 2], [12, 16], k[:28], k[:28])
    assert c.seq_len(0, 1) == 32 and c.seq_len(0, 2) == 16


def test_truncate_gives_the_same_blocks_again(KV):
    from vortex_b200 import _native as N
    H, D, bs = 2, 64, 16
    c = make(KV, 2, H, D, bs, 64, 4)
    k = [rnd((90, H, D), s) for s in range(4)]
    for layer in range(2):
        c.append_chunks(layer, [5, 6], [40, 21], k[layer][:61], k[layer + 2][:61])
    tables = {(l, s): c.block_table(l, s) for l in range(2) for s in (5, 6)}
    free = c.free_block_count()
    for cut5, cut6 in ((17, 21), (16, 0), (0, 1), (39, 20)):
        c.truncate([5, 6, 77], [cut5, cut6, 3])
        assert [c.seq_len(1, s) for s in (5, 6)] == [cut5, cut6]
        assert c.pages()["lens"][:, :2].tolist() == [[cut5, cut6]] * 2
        assert c.free_block_count() == free + 2 * (3 - -(-cut5 // bs) + 2 - -(-cut6 // bs))
        for layer in range(2):
            kk = torch.cat([k[layer][cut5:40], k[layer][40 + cut6:61]])
            vv = torch.cat([k[layer + 2][cut5:40], k[layer + 2][40 + cut6:61]])
            c.append_chunks(layer, [5, 6], [40 - cut5, 21 - cut6], kk, vv)
        assert {t: c.block_table(*t) for t in tables} == tables and c.free_block_count() == free
        for layer in range(2):
            for s, at, n in ((5, 0, 40), (6, 40, 21)):
                gk, gv = c.get_kv(layer, s)
                assert torch.equal(gk, k[layer][at:at + n].float()) and torch.equal(gv, k[layer + 2][at:at + n].float())
    c.truncate([5], [1000])
    assert c.seq_len(0, 5) == 40
    for ids, lens in (([5, 5], [1, 1]), ([5], [-1]), ([5], [1, 2])):
        with pytest.raises(N.VxbError):
            c.truncate(ids, lens)


@pytest.mark.parametrize("int8", [False, True])
def test_truncate_inside_a_shared_block_moves_it(KV, int8):
    H, D, bs = 2, 64, 16
    c = make(KV, 2, H, D, bs, 12, 4, int8)
    k = rnd((48, H, D), 0)
    for layer in range(2):
        c.append_chunks(layer, [0], [40], k[:40], -k[:40])
    c.fork(0, 1, 32)
    want = [c.get_kv(l, 1) for l in range(2)]
    c.truncate([0], [21])  # block 1 is the fork's too
    for layer in range(2):
        assert c.block_table(layer, 0)[1] != c.block_table(layer, 1)[1]
        c.append_chunks(layer, [0], [5], k[40:45], k[40:45])
    for layer in range(2):
        gk, gv = c.get_kv(layer, 1)
        assert torch.equal(gk, want[layer][0]) and torch.equal(gv, want[layer][1])
        gk, gv = c.get_kv(layer, 0)
        assert gk.shape[0] == 26 and torch.equal(gk[:21], want[layer][0][:21]) and torch.equal(gv[:21], want[layer][1][:21])
    c.free_seq(0)
    c.free_seq(1)
    assert c.used_blocks() == 0


# ---------------------------------------------------------------- chunk attention

def stored(c, layer, s):
    k, v = c.get_kv(layer, s)
    return k.double(), v.double()


def exact_rows(q, k, v, m, causal, scale, far=False):
    """out, lse and the two tolerances of the m rows q [m, Hq, D] over k, v [len, Hkv, D] (64 bits)."""
    n, hkv, D = k.shape
    G = q.shape[1] // hkv
    k, v = (t.repeat_interleave(G, 1) for t in (k, v))
    q = q.double()
    s = torch.einsum("mhd,nhd->mhn", q, k) * scale
    last = torch.arange(m, device=q.device) + (n - m) if causal else torch.full((m,), n - 1, device=q.device)
    sees = torch.arange(n, device=q.device)[None] <= last[:, None]
    s = s.masked_fill(~sees[:, None], -math.inf)
    lse = torch.logsumexp(s, -1) if n else torch.full((m, q.shape[1]), -math.inf, device=q.device, dtype=torch.float64)
    p = torch.exp(s - lse[..., None]).nan_to_num(0.0)
    out, a = torch.einsum("mhn,nhd->mhd", p, v), torch.einsum("mhn,nhd->mhd", p, v.abs())
    b = (torch.einsum("mhd,nhd->mhn", q.abs(), k.abs()) * scale).masked_fill(~sees[:, None], 0.0)
    b = b.amax(-1) if n else torch.zeros_like(lse)
    extra = 2 * D * 2.0 ** -24 * b + 2.0 ** -20
    tol = 2.0 ** -8 * out.abs() + (2.0 ** -8 + extra[..., None]) * (1 + 2.0 ** -8) * a
    if far and n:
        # int8 caches whose V scales lie far apart: a weight p_k s_k (s_k the V scale) is kept as f16 in a unit in which
        # the row's largest is 2^6 or more, so below 2^-14 it is off by half of f16's least step, 2^-25: by
        # 2^-31 max(p s). It multiplies a code of at most 127, and max |v_k| = 127 s_k: n 2^-31 max(p_k max |v_k|) in all.
        tol = tol + n * 2.0 ** -31 * (p * v.abs().amax(-1).transpose(0, 1)[None]).amax(-1)[..., None]
    return out, lse, tol, extra + 2.0 ** -22 * lse.abs()


def check_rows(out, lse, q, c, layer, ids, counts, causal, scale, far=False):
    at = 0
    for s, m in zip(ids, counts):
        k, v = stored(c, layer, s)
        o, z, to, tz = exact_rows(q[at:at + m], k, v, m, causal, scale, far)
        g, y = out[at:at + m].double(), lse[at:at + m].double()
        none = torch.isinf(z)
        assert torch.equal(torch.isinf(y) & (y < 0), none), s
        assert bool((g[none] == 0).all()), s
        bad = ((g - o).abs() > to + 1e-30)
        assert not bool(bad.any()), (s, float(((g - o).abs() - to)[bad].max()), bad.nonzero()[:4].tolist())
        dz = (y - z)[~none].abs()
        assert bool((dz <= tz[~none]).all()), (s, float(dz.max()))
        at += m


CHUNKS = [
    # H kv, G, D, block, layers, lens, counts
    (1, 1, 128, 16, [1], [1]),
    (2, 4, 128, 16, [5, 300], [5, 1]),
    (2, 1, 64, 16, [17, 128, 129, 1000], [4, 128, 1, 100]),
    (1, 3, 128, 32, [77, 0, 255, 256], [50, 0, 3, 128]),
    (4, 8, 64, 16, [640, 15], [33, 15]),
    (2, 16, 128, 48, [200, 1500], [9, 2]),
    (1, 128, 64, 16, [40, 130], [3, 1]),
    (3, 5, 128, 64, [513, 700, 64], [257, 61, 64]),
    (2, 2, 128, 16, [2500], [700]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H,G,D,bs,lens,counts", CHUNKS)
def test_chunk_attention_vs_f64(KV, H, G, D, bs, lens, counts, int8, causal):
    n = len(lens)
    c = make(KV, 2, H, D, bs, sum(-(-x // bs) for x in lens) + 3, n + 1, int8)
    c.append_chunks(0, [99], [3], rnd((3, H, D), 9), rnd((3, H, D), 9))  # block 0 is another layer's
    k, v = rnd((sum(lens), H, D), 1), rnd((sum(lens), H, D), 2)
    ids = [10 + i for i in range(n)]
    c.append_chunks(1, ids, lens, k, v)
    q = rnd((sum(counts), H * G, D), 3, 2.0)
    lse = torch.full((sum(counts), H * G), 7.0, device="cuda")
    out = c.chunk_attention(1, ids, counts, q, causal=causal, lse=lse)
    check_rows(out, lse, q, c, 1, ids, counts, causal, 1 / math.sqrt(D))
    assert torch.equal(out, c.chunk_attention(1, ids, counts, q, causal=causal)), "not deterministic"


FEW = [
    # H kv, G, block, lens, counts: up to 64 rows a head, short and long, many and few sequences
    (1, 1, 16, [128 * i + 1 for i in range(20)], [1 + i % 16 for i in range(20)]),
    (4, 4, 16, [3000, 127, 128, 129, 5000], [4, 8, 16, 1, 5]),
    (2, 8, 32, [40, 9000], [8, 8]),
    (1, 64, 16, [700, 31], [1, 1]),
    (1, 24, 128, [2000, 2, 640], [2, 2, 1]),
    (3, 7, 16, [255, 1, 400, 256, 17, 1030], [9, 1, 2, 0, 4, 3]),
    (8, 1, 64, [600] * 40, [64, 1, 3, 33] * 10),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,G,bs,lens,counts", FEW)
def test_chunk_attention_few_rows(KV, H, G, bs, lens, counts, D, int8, causal):
    n = len(lens)
    c = make(KV, 1, H, D, bs, sum(-(-x // bs) for x in lens), n, int8)
    v = rnd((sum(lens), H, D), 2)
    v[::5] *= 100.0  # scales of an int8 cache that differ from key to key
    v[1::7] *= 0.001
    c.append_chunks(0, range(n), lens, rnd((sum(lens), H, D), 1), v)
    q = rnd((sum(counts), H * G, D), 3, 2.0)
    lse = torch.full((sum(counts), H * G), 7.0, device="cuda")
    out = c.chunk_attention(0, range(n), counts, q, causal=causal, lse=lse)
    check_rows(out, lse, q, c, 0, range(n), counts, causal, 1 / math.sqrt(D))
    assert torch.equal(out, c.chunk_attention(0, range(n), counts, q, causal=causal)), "not deterministic"


RUNS = [
    # H kv, G, block, lens, counts: few items of many key tiles, which are cut, and many of few, several to a run
    (1, 4, 16, [2500], [300]),
    (2, 3, 16, [2300, 130, 4000], [100, 90, 60]),
    (1, 1, 32, [1500, 3100, 7], [129, 300, 5]),
    (1, 128, 64, [1900], [5]),
    (8, 1, 16, [130 + 29 * i for i in range(20)], [70 + 13 * (i * 7 % 20) for i in range(20)]),
    (4, 2, 16, [65 + 40 * i for i in range(16)], [65 + 3 * i for i in range(16)]),
    (8, 4, 16, [100 + 33 * (i * 5 % 33) for i in range(33)], [1 + i % 16 for i in range(33)]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,G,bs,lens,counts", RUNS)
def test_chunk_attention_cut_and_whole_runs(KV, H, G, bs, lens, counts, D, int8, causal):
    n = len(lens)
    c = make(KV, 1, H, D, bs, sum(-(-x // bs) for x in lens), n, int8)
    c.append_chunks(0, range(n), lens, rnd((sum(lens), H, D), 1), rnd((sum(lens), H, D), 2))
    q = rnd((sum(counts), H * G, D), 3, 2.0)
    lse = torch.full((sum(counts), H * G), 7.0, device="cuda")
    out = c.chunk_attention(0, range(n), counts, q, causal=causal, lse=lse)
    check_rows(out, lse, q, c, 0, range(n), counts, causal, 1 / math.sqrt(D))
    assert torch.equal(out, c.chunk_attention(0, range(n), counts, q, causal=causal)), "not deterministic"


@pytest.mark.parametrize("m", [150, 60, 24, 5])
@pytest.mark.parametrize("D", [64, 128])
def test_chunk_attention_int8_scales_far_apart(KV, D, m):
    # values near the least and the largest that bf16 holds beside ordinary ones, and keys alike
    H, n = 2, 700
    k, v, q = rnd((n, H, D), 1), rnd((n, H, D), 2), rnd((m, H, D), 3)
    v[3::7] *= 1e-39
    v[5::11] *= 1e-20
    v[n - 2:, 1] *= 1e30
    k[2::9] *= 1e-39
    c = make(KV, 1, H, D, 16, 50, 1, True)
    c.append_chunks(0, [0], [n], k, v)
    lse = torch.zeros(m, H, device="cuda")
    out = c.chunk_attention(0, [0], [m], q, lse=lse)
    check_rows(out, lse, q, c, 0, [0], [m], True, 1 / math.sqrt(D), far=True)


@pytest.mark.parametrize("m", [200, 64])
def test_chunk_attention_non_finite_values_in_cut_items(KV, m):
    H, n, D = 1, 2600, 128  # the chunk's own keys end far behind the first cut
    k, v, q = rnd((n, H, D), 1), rnd((n, H, D), 2), rnd((m, H, D), 3)
    outs = []
    for poison in (False, True):
        c = make(KV, 1, H, D, 16, 170, 1)
        vv = v.clone()
        if poison:
            vv[n - 40, 0, 5] = float("nan")
        c.append_chunks(0, [0], [n], k, vv)
        outs.append(c.chunk_attention(0, [0], [m], q))
    clean, dirty = outs
    assert torch.equal(clean[:m - 40], dirty[:m - 40])
    assert torch.equal(clean[..., 6:], dirty[..., 6:]) and bool(torch.isnan(dirty[m - 40:, 0, 5]).all())


@pytest.mark.parametrize("int8", [False, True])
def test_chunk_attention_rows_that_see_nothing(KV, int8):
    # empty and unknown sequences, more queries than tokens, sequences without queries
    H, D = 2, 128
    c = make(KV, 1, H, D, 16, 32, 8, int8)
    c.append_chunks(0, [1, 2, 3], [3, 150, 16], rnd((169, H, D), 1), rnd((169, H, D), 2))
    c.truncate([3], [0])
    ids, counts = [1, 4, 3, 2, 1], [9, 5, 2, 140, 0]
    q = rnd((sum(counts), 4, D), 3)
    for causal in (True, False):
        lse = torch.zeros(sum(counts), 4, device="cuda")
        out = c.chunk_attention(0, ids, counts, q, causal=causal, lse=lse)
        check_rows(out, lse, q, c, 0, ids, counts, causal, 1 / math.sqrt(D))
    # the same sequence twice is two independent readings of it
    out = c.chunk_attention(0, [2, 2], [140, 140], torch.cat([q[16:156], q[16:156]]))
    assert torch.equal(out[:140], out[140:])
    assert c.chunk_attention(0, [], [], q[:0]).shape == (0, 4, D)
    assert c.chunk_attention(0, [1, 2], [0, 0], q[:0]).shape == (0, 4, D)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("m", [200, 64])
def test_chunk_attention_masked_tokens_do_not_matter(KV, D, m, bad):
    # a later token of the same chunk with a non-finite key or value changes
    # no earlier row; a finite softmax sees only visible tokens
    H, n = 2, 300
    k, v = rnd((n, H, D), 1), rnd((n, H, D), 2)
    q = rnd((m, H, D), 3)
    outs = []
    for poison in (False, True):
        c = make(KV, 1, H, D, 16, 32, 1)
        kk, vv = k.clone(), v.clone()
        if poison:
            kk[250, 1], vv[251, 0, 5], vv[260, 1] = bad, bad, -bad
        c.append_chunks(0, [0], [n], kk, vv)
        outs.append(c.chunk_attention(0, [0], [m], q))
    clean, dirty = outs
    at = n - m                                              # the first row's token
    assert torch.equal(clean[:250 - at], dirty[:250 - at])
    assert torch.equal(clean[:251 - at, 0], dirty[:251 - at, 0])
    assert torch.equal(clean[251 - at:, 0, 6:], dirty[251 - at:, 0, 6:])  # one dimension of one value row
    assert not bool(torch.isfinite(dirty[251 - at:, 0, 5]).any())
    assert not bool(torch.isfinite(dirty[260 - at:, 1]).any())


def test_chunk_attention_many_sequences_streams_and_graphs(KV):
    H, G, D, n = 1, 2, 64, 300
    lens, counts = [1 + (37 * i) % 90 for i in range(n)], [(i * 5) % 4 for i in range(n)]
    c = make(KV, 1, H, D, 16, 6 * n, n)
    c.append_chunks(0, range(n), lens, rnd((sum(lens), H, D), 1), rnd((sum(lens), H, D), 2))
    q = rnd((sum(counts), H * G, D), 3, 2.0)
    lse = torch.empty(sum(counts), H * G, device="cuda")
    want = c.chunk_attention(0, range(n), counts, q, lse=lse)
    check_rows(want, lse, q, c, 0, range(n), counts, True, 1 / math.sqrt(D))
    torch.cuda.synchronize()
    # two calls at once on their own streams
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:
        with torch.cuda.stream(s):
            got.append([c.chunk_attention(0, range(n), counts, q) for _ in range(8)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for g in got for x in g)
    # strided queries, and an output given
    wide = torch.empty(q.shape[0], H * G, 2 * D, dtype=torch.bfloat16, device="cuda")
    wide[..., :D] = q
    out = torch.empty_like(q)
    assert c.chunk_attention(0, range(n), counts, wide[..., :D], out=out) is out and torch.equal(out, want)
    # captured twice, replayed in turn with new queries
    graphs, bufs = [], []
    for _ in range(2):
        qq, oo = q.clone(), torch.empty_like(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.chunk_attention(0, range(n), counts, qq, out=oo)
        graphs.append(g)
        bufs.append((qq, oo))
    bufs[1][0].neg_()
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(bufs[0][1], want) and torch.equal(bufs[1][1], c.chunk_attention(0, range(n), counts, -q))


def test_chunk_attention_refuses(KV):
    from vortex_b200 import _native as N
    c = make(KV, 1, 2, 64, 16, 8, 2)
    c.append_chunks(0, [0], [20], rnd((20, 2, 64), 1), rnd((20, 2, 64), 2))
    q = rnd((4, 6, 64), 3)
    ok = dict(layer=0, seq_ids=[0], n_queries=[4], q=q)
    c.chunk_attention(**ok)
    for change in (dict(layer=1), dict(layer=-1), dict(n_queries=[3]), dict(n_queries=[-4]), dict(seq_ids=[0, 1]), dict(q=q[:, :5]),
                   dict(q=q.float()), dict(q=q[..., :32]), dict(q=q.cpu()), dict(q=q[0]), dict(softmax_scale=0.0),
                   dict(softmax_scale=float("nan")), dict(softmax_scale=float("inf")), dict(out=torch.empty_like(q).float()),
                   dict(out=torch.empty(4, 6, 128, device="cuda", dtype=torch.bfloat16)[..., :64]),
                   dict(lse=torch.empty(4, 5, device="cuda")), dict(q=rnd((4, 258, 64), 1))):
        with pytest.raises(N.VxbError):
            c.chunk_attention(**{**ok, **change})
    import ctypes
    ids, cnt = np.zeros(1, np.int64), np.full(1, 4, np.int32)
    call = lambda ws, n: N.lib().vxb_chunk_attention(c.ptr, 0, 1, ids.ctypes.data, cnt.ctypes.data, q.data_ptr(), 6, 1.0, 1,
                                                     q.data_ptr(), None, ws, n, None)
    need = ctypes.c_size_t()
    assert N.lib().vxb_chunk_attention_ws(c.ptr, 6, ctypes.byref(need)) == 0
    ws = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    assert call(None, need.value) == call(ws.data_ptr(), need.value - 1) == call(ws.data_ptr() + 4, need.value) == N.VXB_EINVAL


def test_chunk_attention_offsets_beyond_32_bits(KV):
    # a pool of more than 2^31 elements: the sequence sits behind them
    H, D, bs = 32, 128, 16
    fill = 2 ** 31 // (H * D) + 64
    c = KV.PagedKVCache(1, H, D, block_size=bs, max_blocks=fill // bs + 80, max_seqs=2, max_blocks_per_seq=fill // bs + 80)
    piece = 65536
    z = torch.zeros(piece, H, D, dtype=torch.bfloat16, device="cuda")
    left = fill
    while left:
        t = min(left, piece)
        c.append_chunks(0, [0], [t], z[:t], z[:t])
        left -= t
    del z
    n, m = 700, 40
    k, v, q = rnd((n, H, D), 1), rnd((n, H, D), 2), rnd((m, H, D), 3, 2.0)
    c.append_chunks(0, [1], [n], k, v)
    assert min(c.block_table(0, 1)) * H * bs * D > 2 ** 31
    lse = torch.empty(m, H, device="cuda")
    out = c.chunk_attention(0, [1], [m], q, lse=lse)
    check_rows(out, lse, q, c, 0, [1], [m], True, 1 / math.sqrt(D))
    # and the long sequence itself, a row over all of it: zeros in, zeros out
    lse = torch.empty(2, H, device="cuda")
    out = c.chunk_attention(0, [0], [2], q[:2], lse=lse)
    assert bool((out == 0).all())
    assert float((lse[:, 0] - torch.tensor([math.log(fill - 1), math.log(fill)], device="cuda")).abs().max()) <= 2 ** -18


# ---------------------------------------------------------------- token probabilities

def check_probs(p, x, t):
    x = x.double()
    m = x.amax(-1, keepdim=True)
    d = (x - m) / t
    want = torch.softmax(x / t, -1)
    d = d.abs().nan_to_num(0.0, posinf=0.0)
    assert bool(((p.double() - want).abs() <= (2.0 ** -17 + 2.0 ** -23 * d) * want + 2.0 ** -125).all())


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (1, 32000), (5, 32001), (40, 1000), (200, 4097), (2, 131072),
                                        (3, 131073), (2, 300007), (161, 20000)])
@pytest.mark.parametrize("t", [0.05, 0.8, 1.0, 30.0])
def test_token_probs_vs_f64(SM, rows, vocab, t):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = 3 * torch.randn(rows, vocab, generator=g, device="cuda")
    if vocab > 3:
        x[:, ::3] = -math.inf
    p = SM.token_probs(x, t)
    check_probs(p, x, t)
    per_row = torch.full((rows,), t, device="cuda")
    assert torch.equal(p, SM.token_probs(x, per_row)) or t not in (1.0, 30.0)
    y = x.clone()
    assert SM.token_probs(y, t, out=y) is y and torch.equal(y, p)
    assert torch.equal(SM.token_probs(x.reshape(rows, 1, vocab), t).reshape(rows, vocab), p)


def test_token_probs_greedy_banned_and_nan_rows(SM):
    for vocab in (7, 5000, 140000):
        x = torch.randn(6, vocab, device="cuda")
        x[0, [2, 5]] = 9.0                # a tie goes to the lowest index
        x[1] = -math.inf                  # nothing allowed
        x[2, 3] = math.nan
        x[3, :-1] = -math.inf             # one token allowed
        t = torch.tensor([0.0, 0.0, 0.005, 0.0, 1.0, -1.0], device="cuda")
        p = SM.token_probs(x, t)
        want = torch.zeros_like(p)
        want[0, 2] = 1
        want[2, x[2].nan_to_num(-math.inf).argmax()] = 1
        want[3, vocab - 1] = 1
        want[5, x[5].argmax()] = 1
        assert torch.equal(p[[0, 1, 2, 3, 5]], want[[0, 1, 2, 3, 5]])
        check_probs(p[4:5], x[4:5], 1.0)
        p = SM.token_probs(x, 1.0)
        assert bool((p[1] == 0).all()) and bool(torch.isnan(p[2]).all()) and float(p[3, -1]) == 1.0 and float(p[3, :-1].sum()) == 0
        assert torch.equal(SM.token_probs(x, 0.0).argmax(-1)[[0, 3]], want[[0, 3]].argmax(-1))


def test_token_probs_refuses(SM):
    from vortex_b200 import _native as N
    x = torch.zeros(2, 8, device="cuda")
    assert SM.token_probs(x[:0]).shape == (0, 8)
    for args in ((x.half(),), (x.cpu(),), (x, float("nan")), (x, float("inf")), (x, torch.ones(3, device="cuda")),
                 (x, torch.ones(2)), (x, 1.0, torch.zeros(2, 9, device="cuda")), (x, 1.0, torch.zeros(8, 2, device="cuda").T),
                 (x[:, :0],)):
        with pytest.raises(N.VxbError):
            SM.token_probs(*args)


# ---------------------------------------------------------------- draft verification

def plain_verify(drafts, counts, p, q, ua, us):
    """The definition, one token at a time, in 64 bits."""
    drafts, p, ua, us = (t.cpu().numpy() for t in (drafts, p, ua, us))
    q = None if q is None else q.cpu().numpy()
    V = p.shape[1]
    tokens, accepted, row, at = [], [], 0, 0
    for i, g in enumerate(counts):
        j = 0
        while j < g:
            t = int(drafts[at + j])
            if not 0 <= t < V or not float(ua[at + j]) * (1.0 if q is None else float(q[at + j, t])) < float(p[row + j, t]):
                break
            j += 1
        pj = p[row + j].astype(np.float64)
        if j < g:
            if q is None:
                qj = np.zeros(V)
                if 0 <= drafts[at + j] < V:
                    qj[drafts[at + j]] = 1.0
            else:
                qj = q[at + j].astype(np.float64)
            left = np.maximum(np.nan_to_num(pj - qj), 0.0)
            if not left.sum() > 0:
                left = np.maximum(np.nan_to_num(pj), 0.0)
        else:
            left = np.maximum(np.nan_to_num(pj), 0.0)
        upto = np.cumsum(left)
        if upto[-1] > 0:
            hits = np.nonzero((upto > float(us[i]) * upto[-1]) & (left > 0))[0]
            drawn = int(hits[0] if hits.size else np.nonzero(left > 0)[0][-1])
        else:
            drawn = 0
        tokens += [int(x) for x in drafts[at:at + j]] + [drawn] + [-1] * (g - j)
        accepted.append(j)
        row, at = row + g + 1, at + g
    return tokens, accepted


@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("vocab,counts", [(1, [0, 1, 3]), (5, [2] * 40), (33, [0, 7, 1]), (1000, [4] * 30), (32000, [5, 0, 3, 8]),
                                          (131072, [1, 2]), (300001, [2]), (50, [1] * 1100), (17, [700])])
def test_verify_drafts_vs_definition(SM, vocab, counts, with_q):
    g = torch.Generator(device="cuda").manual_seed(vocab + len(counts))
    D, n = sum(counts), len(counts)
    logits = 2.0 * torch.randn(D + n, vocab, generator=g, device="cuda")
    p = torch.softmax(logits, -1)
    own = torch.arange(D, device="cuda") + torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor(counts, device="cuda"))
    q = torch.softmax(logits[own] + 0.5 * torch.randn(D, vocab, generator=g, device="cuda"), -1)
    drafts = torch.multinomial(q, 1, generator=g)[:, 0].int() if D else torch.zeros(0, dtype=torch.int32, device="cuda")
    for seed in range(3):
        ua, us = torch.rand(D, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
        if seed == 1:
            ua, us = ua * 0.3, us * 0
        if seed == 2:
            us = 1 - us * 2.0 ** -24
        tokens, accepted = SM.verify_drafts(drafts, counts, p, q if with_q else None, ua, us.clamp(max=1 - 2.0 ** -24))
        want = plain_verify(drafts, counts, p, q if with_q else None, ua, us.clamp(max=1 - 2.0 ** -24))
        assert accepted.tolist() == want[1] and tokens.tolist() == want[0]


def test_verify_drafts_edges(SM):
    # ties on the border, drafts out of range, rows without mass, p == q, NaN
    V = 8
    p = torch.zeros(9, V, device="cuda")
    p[0, 2], p[0, 4] = 0.5, 0.5            # request 0: no drafts, u on the border: the next index
    p[1] = 0.125                           # request 1: draft -1
    p[3] = 0.125                           # request 2: draft V
    p[5, 3] = 1.0                          # request 3: q equals p, u q < p
    p[6] = 0.0                             # its last row has no mass
    p[7, 1], p[7, 6] = math.nan, 0.25      # request 4: a refused draft, NaN beside
    q = torch.zeros(4, V, device="cuda")
    q[0], q[1], q[2, 3], q[3, 5] = 0.125, 0.125, 1.0, 1.0
    drafts = torch.tensor([-1, V, 3, 5], dtype=torch.int32, device="cuda")
    counts = [0, 1, 1, 1, 1]
    ua = torch.tensor([0.0, 0.0, 1 - 2.0 ** -24, 0.5], device="cuda")
    us = torch.tensor([0.5, 0.5, 0.125, 0.7, 0.9], device="cuda")
    for qq in (q, None):
        tokens, accepted = SM.verify_drafts(drafts, counts, p, qq, ua, us)
        want = plain_verify(drafts, counts, p, qq, ua, us)
        assert (tokens.tolist(), accepted.tolist()) == want
    assert tokens.tolist()[0] == 4


def test_verify_drafts_refuses(SM):
    from vortex_b200 import _native as N
    p, q, u = torch.full((5, 8), 0.125, device="cuda"), torch.full((3, 8), 0.125, device="cuda"), torch.zeros(3, device="cuda")
    d = torch.zeros(3, dtype=torch.int32, device="cuda")
    ok = [d, [1, 2], p, q, u, u[:2]]
    SM.verify_drafts(*ok)
    for at, bad in ((0, d[:2]), (0, d.long()), (0, d.cpu()), (1, [1, 1]), (1, [4, -1]), (2, p[:4]), (2, p.double()), (2, p[:, :0]),
                    (3, q[:, :7]), (3, q.half()), (4, u[:2]), (5, u), (4, u.cpu())):
        args = list(ok)
        args[at] = bad
        with pytest.raises(N.VxbError):
            SM.verify_drafts(*args)
    tokens, accepted = SM.verify_drafts(d[:0], [], p[:0], None, u[:0], u[:0])
    assert tokens.numel() == 0 and accepted.numel() == 0


# ---------------------------------------------------------------- together

def test_speculative_steps_together(KV, SM):
    """Append drafts, attend, logits, probabilities, verify, take the refused
    tokens back: the cache then holds what appending the accepted tokens alone
    gives, and every step's tokens are the definition's."""
    H, G, D, V, n = 2, 2, 64, 300, 5
    Hq = H * G
    g = torch.Generator(device="cuda").manual_seed(5)
    emb = torch.randn(V, D, generator=g, device="cuda")
    wk, wv = (torch.randn(D, H * D, generator=g, device="cuda") / 8 for _ in range(2))
    wq, wo = torch.randn(D, Hq * D, generator=g, device="cuda") / 8, torch.randn(Hq * D, V, generator=g, device="cuda") / 4

    def kvq(tok):
        e = emb[tok.long()]
        return ((e @ wk).reshape(-1, H, D).bfloat16(), (e @ wv).reshape(-1, H, D).bfloat16(), (e @ wq).reshape(-1, Hq, D).bfloat16())

    c, plain = (make(KV, 1, H, D, 16, 64, n) for _ in range(2))
    ids = np.arange(n)
    prompt = [torch.randint(0, V, (m,), generator=g, device="cuda") for m in (1, 17, 40, 16, 33)]
    k, v, _ = kvq(torch.cat(prompt))
    for x in (c, plain):
        x.append_chunks(0, ids, [len(t) for t in prompt], k, v)
    held = [len(t) for t in prompt]
    last = torch.stack([t[-1] for t in prompt]).int()
    for step in range(4):
        counts = [(step + i) % 4 for i in range(n)]
        drafts = torch.randint(0, V, (sum(counts),), generator=g, device="cuda").int()
        chunk = torch.cat([torch.cat([last[i:i + 1], d]) for i, d in enumerate(drafts.split(counts))])
        m = [x + 1 for x in counts]
        k, v, q = kvq(chunk)
        c.append_chunks(0, ids, m, k, v)
        lse = torch.empty(sum(m), Hq, device="cuda")
        out = c.chunk_attention(0, ids, m, q, lse=lse)
        check_rows(out, lse, q, c, 0, ids, m, True, 1 / math.sqrt(D))
        p = SM.token_probs(out.float().reshape(-1, Hq * D) @ wo, 0.9)
        ua, us = torch.rand(sum(counts), generator=g, device="cuda") * 2.0 ** -5, torch.rand(n, generator=g, device="cuda")
        tokens, accepted = SM.verify_drafts(drafts, counts, p, None, ua, us)
        assert (tokens.tolist(), accepted.tolist()) == plain_verify(drafts, counts, p, None, ua, us)
        acc = accepted.tolist()
        c.truncate(ids, [h + 1 + a for h, a in zip(held, acc)])
        at, rows = 0, []
        for i in range(n):
            rows.append(torch.arange(at, at + 1 + acc[i]))
            at += m[i]
        rows = torch.cat(rows).cuda()
        plain.append_chunks(0, ids, [1 + a for a in acc], k[rows], v[rows])
        held = [h + 1 + a for h, a in zip(held, acc)]
        last = torch.stack([t[a] for t, a in zip(tokens.split(m), acc)])
        assert c.stats() == plain.stats()
        for i in range(n):
            assert c.block_table(0, i) == plain.block_table(0, i)
            for x, y in zip(c.get_kv(0, i), plain.get_kv(0, i)):
                assert torch.equal(x, y)
    # a decode step reads the same cache
    qq = rnd((n, Hq, D), 8)
    assert torch.equal(c.attention(0, ids, qq), plain.attention(0, ids, qq))


@pytest.mark.parametrize("int8", [False, True])
def test_pages_behind_four_gigabytes(KV, int8):
    H, D, bs = 32, 128, 1024
    fill = 1100 if int8 else 560  # sequences of one token, each with a block of its own
    c = make(KV, 1, H, D, bs, fill + 4, fill + 1, int8)
    one = rnd((fill, H, D), 0)
    c.append_chunks(0, range(fill), [1] * fill, one, one)
    n = 2500
    c.append_chunks(0, [fill], [n], rnd((n, H, D), 1), rnd((n, H, D), 2))
    assert min(c.block_table(0, fill)) * H * bs * D * (1 if int8 else 2) > 2 ** 32
    for m in (3, 200):
        q, lse = rnd((m, H, D), 3, 2.0), torch.empty(m, H, device="cuda")
        out = c.chunk_attention(0, [fill], [m], q, lse=lse)
        check_rows(out, lse, q, c, 0, [fill], [m], True, 1 / math.sqrt(D))
    assert torch.equal(c.get_kv(0, 7)[0][0], c.get_kv(0, 7)[1][0])
    c.truncate([fill], [n - 40])
    assert c.pages()["lens"][0, fill].item() == n - 40


@pytest.mark.parametrize("int8", [False, True])
def test_calls_in_a_row_without_waiting(KV, int8):
    # each call starts while the last may still run: appends, attention whose
    # items are cut and joined, and few rows, all over one scratch allocator
    H, G, D, lens = 1, 4, 128, [2000, 700]
    c = make(KV, 1, H, D, 16, 300, 2, int8)
    c.append_chunks(0, [0, 1], lens, rnd((sum(lens), H, D), 1), rnd((sum(lens), H, D), 2))
    torch.cuda.synchronize()
    got = []
    for step, counts in enumerate([[200, 3], [5, 1], [1, 140], [70, 70], [2, 2], [300, 0]]):
        k, v = rnd((sum(counts), H, D), 10 + step), rnd((sum(counts), H, D), 20 + step)
        q, lse = rnd((sum(counts), H * G, D), 30 + step, 2.0), torch.empty(sum(counts), H * G, device="cuda")
        c.append_chunks(0, [0, 1], counts, k, v)
        got.append((counts, q, c.chunk_attention(0, [0, 1], counts, q, lse=lse), lse))
    total = [a + sum(x[0][i] for x in got) for i, a in enumerate(lens)]
    for counts, q, out, lse in got[::-1]:
        c.truncate([0, 1], total)
        check_rows(out, lse, q, c, 0, [0, 1], counts, True, 1 / math.sqrt(D))
        total = [a - b for a, b in zip(total, counts)]


def test_probabilities_of_too_large_a_vocabulary_are_refused(SM):
    from vortex_b200 import _native as N
    from vortex_b200.quant import context
    ctx, x = context(0), torch.zeros(8, device="cuda")
    with pytest.raises(N.VxbError) as e:
        ctx.call("vxb_token_probs", x.data_ptr(), 1, 2 ** 30 + 1, None, 1.0, x.data_ptr(), None)
    assert e.value.code == N.VXB_EUNSUPPORTED
    with pytest.raises(N.VxbError) as e:
        ctx.call("vxb_verify_drafts", 1, np.zeros(1, np.int32).tobytes(), 2 ** 30 + 1, None, x.data_ptr(), None, None,
                 x.data_ptr(), x.data_ptr(), x.data_ptr(), None)
    assert e.value.code == N.VXB_EUNSUPPORTED
