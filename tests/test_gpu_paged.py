"""Caches in pages: appends against the contiguous ones byte for byte, loads and attention against 64 bits.

Tolerance of the attention (rows of 128 outputs, 2-norm).  Besides the output's own rounding (eps / 2 of it): weights and rotated
queries are rounded to fp16 (2^-11 each, independent from place to place), which moves a row by the root of the sum of squares of
weight x |value| x (2^-11 + the logit's error), the logit's error being 2^-11 x scale x the root of sum (q_i k_i)^2; four times
that is allowed.  Codebooks and 8-bit values are rounded to fp16 once for all places, at most 2^-11 on either side: 2^-10 of the
output.  32-bit sums lose 2^-20 of sum weight |value|.
"""
import numpy as np
import pytest

import turboquant_plus_amd as tqa
from turboquant_plus_amd import _lib as L
from turboquant_plus_amd.turbo import OVERRUN_NEGATIVE, OVERRUN_NO_ROOM, overrun_bits
from turboquant_plus_amd.paged import OVERRUN_NO_PAGE

pytestmark = pytest.mark.gpu
tt = L.torch()
D = 128
FORMATS = ("turbo2", "turbo3", "turbo4", "q8_0")
DTYPES = {"fp16": tt.float16, "bf16": tt.bfloat16, "fp32": tt.float32}


def layer(k, v):
    return tqa.LayerKV(tqa.LayerFormat(k, v), seed=7)


def ints(x):
    return tt.tensor(x, dtype=tt.int32, device="cuda")


def cumulative(n):
    return ints(np.concatenate([[0], np.cumsum(n)]).tolist())


def table_for(lens, n_pages, seed=0, width=None):
    """Distinct random pages for every sequence; entries that no token needs are no pages at all."""
    blocks = [-(-c // 128) for c in lens]
    t = np.full((len(lens), max(max(blocks), width or 1)), -1, np.int32)
    free = np.random.default_rng(seed).permutation(n_pages)[:sum(blocks)]
    assert len(free) == sum(blocks)
    for b, n in enumerate(blocks):
        t[b, :n], free = free[:n], free[n:]
    return ints(t.tolist())


def outliers(x):
    x[..., ::37] *= 12
    return x


def values(codec, pages, kind):
    """[pages, heads, 128 tokens, 128] in 64 bits, turbo rows in the rotated domain, by the reference decoders."""
    n, h, _ = pages.shape
    if codec is None:
        q, s = tqa.q8_0_unpack(pages.reshape(-1), n * h, 128, kind)
        return (q.double().view(n, h, 128, 4, 32) * s.double().view(n, h, 128, 4, 1)).view(n, h, 128, D)
    idx, norm = codec.unpack_codes(pages.reshape(-1), n * h, 128, kind)
    return tt.tensor(codec.centroids, device="cuda")[idx.long()].view(n, h, 128, D) * norm.double().view(n, h, 128, 1)


def rotation(codec):
    """R of y = R x, in 64 bits."""
    i = np.arange(D)
    H = 1 - 2 * (np.vectorize(lambda x: bin(x).count("1") & 1)(i[:, None] & i[None]))
    return tt.tensor(codec.signs2[:, None] * H * codec.signs1[None] / np.sqrt(D), device="cuda")


def attend64(lay, q, kp, vp, table, lens, new, causal, scale=D ** -0.5):
    """(out, allowed error of each row) in 64 bits, row by row of the batch."""
    k, v = values(lay.k_codec, kp, "k"), values(lay.v_codec, vp, "v")
    hkv, hq = kp.shape[1], q.shape[1]
    g, out, tol, at = hq // hkv, tt.zeros(q.shape, dtype=tt.float64, device="cuda"), tt.zeros(q.shape[:2], dtype=tt.float64, device="cuda"), 0
    eps = tt.finfo(q.dtype).eps
    for b, (n, c) in enumerate(zip(new, lens)):
        pages = table[b, :-(-c // 128)].long()
        x = q[at:at + n].double()
        if lay.k_codec is not None:
            x = x @ rotation(lay.k_codec).T
        seen = tt.arange(c, device="cuda")[None] < (c - n + tt.arange(n, device="cuda")[:, None] + 1 if causal else c)
        seen = seen.expand(n, c).repeat_interleave(g, 0)
        for h in range(hkv):
            kk, vv = k[pages, h].reshape(-1, D)[:c], v[pages, h].reshape(-1, D)[:c]
            xx = x[:, h * g:(h + 1) * g].reshape(-1, D)
            logits = scale * xx @ kk.T
            w = tt.softmax(tt.where(seen, logits, -float("inf")), -1).nan_to_num(0.0) if c else tt.zeros((n * g, 0), device="cuda").double()
            y = w @ vv
            off = 2 ** -11 * (1 + scale * (xx.square() @ kk.square().T).sqrt())
            size = vv.norm(dim=-1)
            tol[at:at + n, h * g:(h + 1) * g] = ((eps / 2 + 2 ** -10) * y.norm(dim=-1) + 4 * (w * size * off).norm(dim=-1) + 2 ** -20 * (w @ size)
                                                 + 2.0 ** -24).view(n, g)
            out[at:at + n, h * g:(h + 1) * g] = (y if lay.v_codec is None else y @ rotation(lay.v_codec)).view(n, g, D)
        at += n
    return out, tol


def check(got, want, tol):
    err = (got.double() - want).norm(dim=-1)
    assert tt.isfinite(got).all()
    assert (err <= tol).all(), (float((err - tol).max()), float((err / tol.clamp(min=1e-30)).max()))


def filled(lay, lens, hkv, seed, extra=2, width=None):
    """Pages with `lens` tokens of every sequence appended."""
    n_pages = sum(-(-c // 128) for c in lens) + extra
    kp, vp = lay.new_pages(n_pages, hkv)
    table = table_for(lens, n_pages, seed, width)
    gen = tt.Generator("cuda").manual_seed(seed)
    k, v = outliers(tt.randn((sum(lens), hkv, D), generator=gen, device="cuda")).half(), tt.randn((sum(lens), hkv, D), generator=gen, device="cuda").half()
    if sum(lens):
        lay.append_paged(k, v, kp, vp, table, ints([0] * len(lens)), cumulative(lens))
    return kp, vp, table


# ---- appends ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kf,vf", [("turbo3", "turbo3"), ("turbo4", "turbo2"), ("turbo2", "turbo4"), ("q8_0", "turbo3"), ("turbo3", "q8_0"), ("q8_0", "q8_0")])
def test_appends_leave_the_bytes_of_contiguous_appends(kf, vf, dtype):
    """Three ragged steps: prompts (one sequence sits out), chunks that begin inside a block, single tokens."""
    lay, hkv, cap = layer(kf, vf), 3, 512
    steps = [(130, 0, 1, 257), (5, 200, 127, 1), (1, 1, 1, 1)]
    lens = np.zeros(4, int)
    n_pages = 16 + 3
    kp, vp = lay.new_pages(n_pages, hkv)
    kp.fill_(0xA5), vp.fill_(0xA5)
    table = table_for([cap] * 4, n_pages, 1)
    refs = [lay.new_cache(hkv, cap) for _ in steps[0]]
    gen = tt.Generator("cuda").manual_seed(2)
    for new in steps:
        k, v = (tt.randn((sum(new) + 2, hkv, D), generator=gen, device="cuda").to(DTYPES[dtype]) for _ in range(2))   # two rows that are nobody's
        out = lay.append_paged(k, v, kp, vp, table, ints(lens.tolist()), cumulative(new))
        assert out[0] is kp and out[1] is vp
        at = 0
        for b, n in enumerate(new):
            if n:
                take = lambda x: (x.float() if dtype == "bf16" else x)[at:at + n].transpose(0, 1).contiguous()
                lay.append(take(k), take(v), *refs[b], int(lens[b]), cap)
            at += n
        lens += new
        for b in range(4):
            for pool, ref in ((kp, refs[b][0]), (vp, refs[b][1])):
                ref = ref.view(hkv, cap // 128, -1)
                for i in range(-(-int(lens[b]) // 128)):
                    assert tt.equal(pool[table[b, i].item()], ref[:, i]), (new, b, i)
    used = {int(table[b, i]) for b in range(4) for i in range(-(-int(lens[b]) // 128))}
    for p in set(range(n_pages)) - used:
        assert (kp[p] == 0xA5).all() and (vp[p] == 0xA5).all()


def test_append_takes_slices_of_a_fused_projection_and_one_row_each():
    lay, hkv = layer("turbo3", "turbo4"), 2
    gen = tt.Generator("cuda").manual_seed(3)
    for dtype, pad in ((tt.float16, 0), (tt.bfloat16, 8), (tt.float32, 1)):        # 1: rows that have to be copied first
        qkv = tt.randn((70, 8 * D + pad), generator=gen, device="cuda").to(dtype)
        k, v = qkv[:, 4 * D:6 * D].unflatten(1, (2, D)), qkv[:, 6 * D:8 * D].unflatten(1, (2, D))
        starts = ints([(37 * b) % 300 for b in range(70)])
        table = table_for([384] * 70, 210, 4)
        pools = [lay.new_pages(210, hkv) for _ in range(2)]
        lay.append_paged(k, v, *pools[0], table, starts)
        lay.append_paged(k.contiguous(), v.contiguous(), *pools[1], table, starts, ints(list(range(71))))
        assert all(tt.equal(a, b) for a, b in zip(*pools)) and bool(pools[0][0].any())


def test_append_refuses_places_and_says_why():
    lay, hkv = layer("turbo3", "q8_0"), 2
    kp, vp = lay.new_pages(4, hkv)
    kp.fill_(1), vp.fill_(1)
    k = tt.ones((6, hkv, D), device="cuda", dtype=tt.float16)
    word = tt.zeros(1, dtype=tt.int32, device="cuda")
    for table, starts, cu, why in [([[0, 1]], [-1], [0, 6], OVERRUN_NEGATIVE), ([[0, 1]], [251], [0, 6], OVERRUN_NO_ROOM), ([[0, 9]], [128], [0, 6], OVERRUN_NO_PAGE),
                                   ([[0, -1]], [128], [0, 6], OVERRUN_NO_PAGE), ([[0, 1]], [0], [0, 7], OVERRUN_NO_PAGE), ([[0, 1]], [0], [-1, 4], OVERRUN_NO_PAGE),
                                   ([[0, 1]], [0], [5, 2], OVERRUN_NO_PAGE), ([[0, 1]], [2 ** 31 - 1], [0, 6], OVERRUN_NO_ROOM)]:
        word.zero_()
        lay.append_paged(k, k, kp, vp, ints(table), ints(starts), ints(cu), overrun=word)
        assert overrun_bits(word) == why, (table, starts, cu)
        lay.append_paged(k, k, kp, vp, ints(table), ints(starts), ints(cu))
        assert (kp == 1).all() and (vp == 1).all()
    # the others of a batch are written, and so is the block that has a page
    word.zero_()
    lay.append_paged(k, k, kp, vp, ints([[0, 1], [2, 77]]), ints([-3, 126]), ints([0, 2, 6]), overrun=word)
    assert overrun_bits(word) == OVERRUN_NEGATIVE | OVERRUN_NO_PAGE
    assert (kp[:2] == 1).all() and (kp[3] == 1).all() and not (kp[2] == 1).all()


@pytest.mark.parametrize("kf", FORMATS)
@pytest.mark.parametrize("vf", FORMATS)
def test_load_gives_back_what_the_pages_hold(kf, vf):
    """Within fp16's half step and the codebook's in fp16 (2^-11 each) of the values in 64 bits; other rows stay."""
    lay, hkv, lens = layer(kf, vf), 2, [300, 64, 1, 513]
    kp, vp, table = filled(lay, lens, hkv, 5)
    starts, new = [65, 0, 0, 127], [235, 64, 1, 130]
    out = tuple(tt.full((sum(new) + 3, hkv, D), 7.0, dtype=tt.float16, device="cuda") for _ in range(2))
    got = lay.load_paged(kp, vp, table, ints(starts), cumulative(new), out=out)
    for x, codec, pool, kind in zip(got, (lay.k_codec, lay.v_codec), (kp, vp), "kv"):
        want = values(codec, pool, kind)
        if codec is not None:
            want = want @ rotation(codec)
        at = 0
        for b, (s, n) in enumerate(zip(starts, new)):
            ref = want[table[b, :-(-lens[b] // 128)].long()].transpose(1, 2).reshape(-1, hkv, D)[s:s + n]
            err = (x[at:at + n].double() - ref).abs()
            size = ref.norm(dim=-1, keepdim=True) / np.sqrt(D)
            bound = 2 ** -11 * ref.abs() + (0 if codec is None else 4 * 2 ** -11 * size) + 2.0 ** -24
            assert (err <= bound).all(), (kind, float((err - bound).max()))
            at += n
        assert (x[at:] == 7).all()
    rows = lay.load_paged(kp, vp, table, ints([0] * 4))
    assert rows[0].shape == (4, hkv, D)


# ---- attention -------------------------------------------------------------------------------------------------------

CASES = [  # query heads, KV heads, contexts, new tokens, causal
    (4, 1, (1,), (1,), True), (8, 2, (63, 64, 65, 500), (1, 1, 1, 1), True), (32, 8, (4000,), (1,), True),
    (16, 1, (129, 1000), (1, 1), True), (24, 1, (200, 77), (1, 1), True), (40, 8, (300, 130, 5), (3, 2, 5), True),
    (4, 4, (700, 128, 33), (700, 128, 33), True), (5, 1, (257, 600), (129, 600), True), (8, 2, (450, 0, 90), (30, 0, 17), False),
    (6, 3, (1, 129), (200, 3), False), (64, 8, (3000, 250), (5, 5), True), (1, 1, (6000,), (40,), True)]


@pytest.mark.parametrize("hq,hkv,lens,new,causal", CASES)
@pytest.mark.parametrize("kf,vf,dtype", [("turbo3", "turbo3", "fp16"), ("turbo4", "turbo2", "bf16"), ("q8_0", "turbo4", "fp16"), ("turbo2", "q8_0", "bf16")])
def test_attention_against_64_bits(kf, vf, dtype, hq, hkv, lens, new, causal):
    lay = layer(kf, vf)
    kp, vp, table = filled(lay, lens, hkv, 11)
    gen = tt.Generator("cuda").manual_seed(12)
    q = tt.randn((sum(new), hq, D), generator=gen, device="cuda").to(DTYPES[dtype])
    want, tol = attend64(lay, q, kp, vp, table, lens, new, causal)
    attn = lay.paged_attention(hq, hkv, causal=causal)
    cu = None if all(n == 1 for n in new) else cumulative(new)
    check(attn(q, kp, vp, table, ints(lens), cu), want, tol)
    got = attn(q, kp, vp, table, ints(lens), cumulative(new), max_context=max(lens), max_new=max(new))
    assert got.dtype == q.dtype and got.is_contiguous()
    check(got, want, tol)


@pytest.mark.parametrize("kf", FORMATS)
@pytest.mark.parametrize("vf", FORMATS)
def test_every_pair_of_formats_at_every_number_of_row_blocks(kf, vf):
    lay, lens = layer(kf, vf), (333, 70)
    kp, vp, table = filled(lay, lens, 2, 13)
    gen = tt.Generator("cuda").manual_seed(14)
    for new in ((4, 3), (7, 2), (40, 70)):      # 16, 28 and 160 rows
        q = tt.randn((sum(new), 8, D), generator=gen, device="cuda").half()
        want, tol = attend64(lay, q, kp, vp, table, lens, new, True)
        check(lay.paged_attention(8, 2)(q, kp, vp, table, ints(lens), cumulative(new), max_new=max(new)), want, tol)


def test_codebooks_of_their_own_and_a_scale():
    """K and V of one width with different centroids (two tables), an asymmetric codebook among them."""
    lay = layer("turbo3", "turbo3")
    lay.v_codec = tqa.TurboCodec(3, seed=507, centroids=np.array([-0.21, -0.12, -0.07, -0.02, 0.03, 0.08, 0.13, 0.2]))
    kp, vp = lay.new_pages(4, 2)
    gen = tt.Generator("cuda").manual_seed(15)
    lens = (250, 131)
    table = ints([[2, 0], [3, 1]])
    for b, n in enumerate(lens):    # an asymmetric codebook has no paged append: blocks of the contiguous one
        x = tt.randn((2, n, D), generator=gen, device="cuda").half()
        pk, pv = (c.store(x, kind=kind).view(2, 2, -1) for c, kind in ((lay.k_codec, "k"), (lay.v_codec, "v")))
        for i in range(2):
            kp[table[b, i]], vp[table[b, i]] = pk[:, i], pv[:, i]
    for new, scale in (((1, 1), 0.3), ((30, 20), 0.02)):
        q = tt.randn((sum(new), 4, D), generator=gen, device="cuda").half()
        want, tol = attend64(lay, q, kp, vp, table, lens, new, True, scale)
        check(lay.paged_attention(4, 2, scale=scale)(q, kp, vp, table, ints(lens), cumulative(new)), want, tol)
    with pytest.raises(NotImplementedError, match="not symmetric"):
        lay.append_paged(q, q, *lay.new_pages(1, 4), ints([[0]]), ints([0]), cumulative([50]))


@pytest.mark.parametrize("kf,vf", [("turbo3", "turbo3"), ("q8_0", "q8_0")])
@pytest.mark.parametrize("new", [1, 5, 100])
def test_what_lies_in_masked_places_does_not_matter(kf, vf, new):
    """Infinities and NaN behind the context, in pages that are nobody's and in later tokens' rows; entries that are no pages."""
    lay, lens = layer(kf, vf), (150, 260)
    kp, vp, table = filled(lay, lens, 2, 16, width=5)
    gen = tt.Generator("cuda").manual_seed(17)
    q = tt.randn((2 * new, 4, D), generator=gen, device="cuda").half()
    attn = lay.paged_attention(4, 2)
    args = ints(lens), cumulative([new, new])
    want = attn(q, kp, vp, table, *args)
    assert tt.isfinite(want).all()
    for pool, codec in ((kp, lay.k_codec), (vp, lay.v_codec)):
        keep = pool.clone()
        pool.fill_(0xFF)        # norms and scales that are NaN
        for b, c in enumerate(lens):
            for i in range(-(-c // 128)):
                p = int(table[b, i])
                pool[p] = keep[p]
                side = pool[p].view(2, -1)[:, 128 * (128 if codec is None else 16 * codec.bits):].view(tt.int16)
                behind = tt.arange(128, device="cuda") >= c - 128 * i
                if codec is not None:
                    side[:, behind] = 0x7C00
                elif pool is kp:
                    side.view(2, 128, 4)[:, behind] = 0x7C00
                else:
                    side.view(2, 2, 4, 64).transpose(2, 3).reshape(2, 128, 4)  # [tile][block][token]
                    side.view(2, 2, 4, 64)[behind.view(1, 2, 1, 64).expand(2, 2, 4, 64)] = 0x7E00
    assert tt.equal(attn(q, kp, vp, table, *args), want)
    # the newest token of sequence 0 holds no numbers: only the row that sees it changes
    bad = tt.full((1, 2, D), float("nan"), device="cuda", dtype=tt.float16)
    lay.append_paged(tt.zeros_like(bad), bad, kp, vp, table[:1], ints([149]), ints([0, 1]))
    got = attn(q, kp, vp, table, *args)
    if new > 1:
        assert tt.equal(got[:new - 1], want[:new - 1])
    assert tt.equal(got[new:], want[new:])
    if vf == "turbo3":
        assert not tt.isfinite(got[new - 1]).any()


@pytest.mark.parametrize("kf,vf", [("turbo4", "turbo4"), ("q8_0", "turbo3"), ("turbo2", "q8_0")])
@pytest.mark.parametrize("new", [1, 3, 7, 12, 16, 40, 80])
def test_a_block_without_a_page_is_not_seen(kf, vf, new):
    """In the middle of a context: the result is that of the other blocks (4 to 320 rows)."""
    lay, c = layer(kf, vf), 3000
    kp, vp, table = filled(lay, (c,), 1, 35)
    gen = tt.Generator("cuda").manual_seed(36)
    q = tt.randn((new, 4, D), generator=gen, device="cuda").half()
    rest = tt.cat([table[:, :3], table[:, 4:9], table[:, 10:]], 1).contiguous()
    want, tol = attend64(lay, q, kp, vp, rest, (c - 256,), (new,), False)
    for none in (-1, kp.shape[0], 2 ** 31 - 1, -2 ** 31):
        holes = table.clone()
        holes[0, 3] = holes[0, 9] = none
        check(lay.paged_attention(4, 1, causal=False)(q, kp, vp, holes, ints([c]), cumulative([new])), want, tol)
    assert (lay.paged_attention(4, 1)(q, kp, vp, table * 0 - 1, ints([c]), cumulative([new])) == 0).all()


@pytest.mark.parametrize("kf,vf", [("turbo4", "turbo4"), ("turbo3", "turbo4"), ("q8_0", "turbo2"), ("turbo2", "q8_0")])
@pytest.mark.parametrize("hq,new", [(32, 1), (64, 1), (32, 2), (32, 9)])
def test_masked_places_of_long_batches(kf, vf, hq, new):
    """The same where workgroups hold several tiles, with 4-bit tables of a copy per lane among them; entries behind the context are no pages."""
    lay, hkv = layer(kf, vf), 8
    lens = [3000 - 37 * b for b in range(24)]
    kp, vp, table = filled(lay, lens, hkv, 33, width=25)
    gen = tt.Generator("cuda").manual_seed(34)
    q = tt.randn((24 * new, hq, D), generator=gen, device="cuda").half()
    call = lambda: lay.paged_attention(hq, hkv)(q, kp, vp, table, ints(lens), cumulative([new] * 24), max_new=new)
    want = call()
    assert tt.isfinite(want).all()
    for pool, codec in ((kp, lay.k_codec), (vp, lay.v_codec)):
        for b, c in enumerate(lens):
            if c % 128:
                side = pool[int(table[b, c // 128])][:, 128 * (128 if codec is None else 16 * codec.bits):].view(tt.int16)
                if codec is not None:
                    side[:, c % 128:] = 0x7E00
                elif pool is kp:
                    side.view(hkv, 128, 4)[:, c % 128:] = 0x7E00
                else:
                    behind = (tt.arange(128, device="cuda") >= c % 128).view(1, 2, 1, 64)
                    side.view(hkv, 2, 4, 64)[behind.expand(hkv, 2, 4, 64)] = 0x7E00
    assert tt.equal(call(), want)


def test_a_query_that_is_no_number_stays_in_its_row():
    lay, lens = layer("turbo3", "turbo4"), (500,)
    kp, vp, table = filled(lay, lens, 1, 18)
    q = tt.randn((20, 4, D), device="cuda").half()
    want = lay.paged_attention(4, 1)(q, kp, vp, table, ints(lens), cumulative([20]))
    q[3, 2, 17], q[9, 0, 5] = float("nan"), float("inf")
    got = lay.paged_attention(4, 1)(q, kp, vp, table, ints(lens), cumulative([20]))
    same = (got == want).all(-1)
    assert not same[3, 2] and not same[9, 0] and int(same.sum()) == 78
    big = (q * 0).nan_to_num(0.0).bfloat16() + 3e30      # a row's size is taken out before fp16
    assert tt.isfinite(lay.paged_attention(4, 1, scale=1e-17)(big, kp, vp, table, ints(lens), cumulative([20]))).all()


@pytest.mark.parametrize("kf,vf", [("turbo3", "turbo3"), ("turbo4", "turbo4"), ("q8_0", "turbo2"), ("turbo2", "q8_0")])
@pytest.mark.parametrize("hq,new,lens", [(4, 1, 500), (8, 1, 5000), (4, 3, 5000), (4, 7, 400), (4, 10, 5000), (4, 40, 300)])
def test_few_rows_that_are_no_numbers_or_huge(kf, vf, hq, new, lens):
    """The same at every number of rows: one and several passes, 28, 40 and 160 rows, joined through memory and not."""
    lay, lens = layer(kf, vf), (lens, 200)
    kp, vp, table = filled(lay, lens, 1, 24)
    gen = tt.Generator("cuda").manual_seed(25)
    q = tt.randn((2 * new, hq, D), generator=gen, device="cuda").half()
    args = kp, vp, table, ints(lens), cumulative([new, new])
    want = lay.paged_attention(hq, 1)(q, *args)
    bad = q.clone()
    bad[0, 1, 17], bad[-1, 3, 5] = float("nan"), float("-inf")
    got = lay.paged_attention(hq, 1)(bad, *args)
    same = (got == want).all(-1)
    assert not tt.isfinite(got[0, 1]).any() and int(same.sum()) >= 2 * new * hq - 2
    if kf != "q8_0":     # a rotated row holds its infinity in every place
        assert not tt.isfinite(got[-1, 3]).any()
    # a row's size is taken out before fp16, and logits that 32 bits hold with steps of many units have a softmax all the same
    for factor, scale in ((1e30, 1e-17), (1e-30, 1e17), (3e20, 1.0)):
        x = (q.float() * factor).bfloat16()
        y, tol = attend64(lay, x, kp, vp, table, lens, [new, new], True, scale)
        out = lay.paged_attention(hq, 1, scale=scale)(x, *args)
        assert tt.isfinite(out).all()
        if factor < 1:
            check(out, y, tol)


@pytest.mark.parametrize("hq,hkv,batch,new,top", [(32, 8, 64, 1, 260), (64, 8, 64, 1, 260), (8, 2, 300, 1, 130), (4, 1, 520, 2, 70), (32, 8, 32, 1, 3000), (64, 8, 16, 2, 3100),
                                                  (2, 2, 5, 1, 9000), (12, 1, 3, 1, 20000)])
@pytest.mark.parametrize("kf,vf,dtype", [("turbo3", "turbo3", "fp16"), ("turbo4", "turbo4", "bf16"), ("turbo4", "turbo3", "fp16"), ("q8_0", "q8_0", "fp16")])
def test_few_rows_of_ragged_batches(kf, vf, dtype, hq, hkv, batch, new, top):
    """Groups that share a workgroup, sequences shorter than a workgroup's part, empty ones, ones without rows, many parts."""
    lay = layer(kf, vf)
    rng = np.random.default_rng(26)
    lens = [int(top if b == batch - 1 else 0 if b % 17 == 3 else rng.integers(1, top + 1)) for b in range(batch)]
    news = [0 if b % 13 == 5 else int(rng.integers(1, new + 1)) for b in range(batch)]
    kp, vp, table = filled(lay, lens, hkv, 27)
    gen = tt.Generator("cuda").manual_seed(28)
    q = tt.randn((sum(news) + 1, hq, D), generator=gen, device="cuda").to(DTYPES[dtype])
    out = tt.full_like(q, 7.0)
    attn = lay.paged_attention(hq, hkv)
    attn(q, kp, vp, table, ints(lens), cumulative(news), max_new=new, out=out)
    assert (out[-1] == 7).all()
    want, tol = attend64(lay, q[:-1], kp, vp, table, lens, news, True)
    check(out[:-1], want, tol)
    again = tt.full_like(q, 7.0)
    attn(q, kp, vp, table, ints(lens), cumulative(news), max_new=new, max_context=top + 1000, out=again)     # another split of the positions
    check(again[:-1], want, tol)


def test_two_captured_steps_of_different_plans_share_a_workspace():
    """Replayed in turn, with eager work between: each finds its counters whatever the other left in them."""
    lay = layer("turbo4", "turbo4")
    lens = (9000, 300, 5000)
    kp, vp, table = filled(lay, lens, 2, 29)
    gen = tt.Generator("cuda").manual_seed(30)
    q = tt.randn((6, 8, D), generator=gen, device="cuda").half()
    attn = lay.paged_attention(8, 2)
    calls = [lambda out: attn(q[:3], kp, vp, table, ints_lens, max_context=9000, out=out),
             lambda out: attn(q, kp, vp, table, ints_lens, cu, max_context=20000, max_new=2, out=out)]
    ints_lens, cu = ints(lens), cumulative([2, 2, 2])
    outs = [tt.empty((n, 8, D), dtype=tt.float16, device="cuda") for n in (3, 6)]
    want = [call(tt.empty_like(out)) for call, out in zip(calls, outs)]
    graphs = []
    side = tt.cuda.Stream()
    with tt.cuda.stream(side):
        for call, out in zip(calls, outs):
            call(out)
            side.synchronize()
            g = tt.cuda.CUDAGraph()
            with tt.cuda.graph(g, stream=side):
                call(out)
            graphs.append(g)
    tt.cuda.synchronize()
    for turn in (0, 1, 0, 0, 1, 1, 0):
        outs[turn].fill_(7.0)
        graphs[turn].replay()
        tt.cuda.synchronize()
        assert tt.equal(outs[turn], want[turn]), turn
        assert tt.equal(calls[1 - turn](tt.empty_like(outs[1 - turn])), want[1 - turn])


def test_a_captured_step_outlives_its_workspace():
    """A larger call replaces the object's workspace; what was captured with the smaller one still has it to itself."""
    lay, lens = layer("turbo3", "turbo3"), (2000,)
    kp, vp, table = filled(lay, lens, 1, 37)
    q = tt.randn((8, 4, D), device="cuda").half()
    n, cu = ints(lens), cumulative([8])
    attn, out = lay.paged_attention(4, 1), tt.empty((1, 4, D), dtype=tt.float16, device="cuda")
    call = lambda: attn(q[:1], kp, vp, table, n, max_context=2000, out=out)
    side = tt.cuda.Stream()
    side.wait_stream(tt.cuda.current_stream())
    with tt.cuda.stream(side):
        call()
        side.synchronize()
        graph = tt.cuda.CUDAGraph()
        with tt.cuda.graph(graph, stream=side):
            call()
    tt.cuda.synchronize()
    want, small = out.clone(), attn.workspace.numel()
    wide = tt.zeros((1, 4000), dtype=tt.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    attn(q, kp, vp, wide, n, cu)        # positions up to 512 000 size it
    assert attn.workspace.numel() > small
    with tt.cuda.stream(side):          # what the allocator may hand out again
        taken = [tt.full((small,), 1, dtype=tt.uint8, device="cuda") for _ in range(4)]
    for _ in range(3):
        out.zero_()
        graph.replay()
        tt.cuda.synchronize()
        assert tt.equal(out, want) and all((x == 1).all() for x in taken)


@pytest.mark.parametrize("causal", [True, False])
def test_rows_that_see_nothing_and_rows_of_nobody(causal):
    lay = layer("turbo3", "turbo2")
    kp, vp, table = filled(lay, (130, 0, 3), 2, 19)
    q = tt.randn((12, 4, D), device="cuda").half()
    for lens in ((130, 0, 3), (0, 0, 0), (-5, 0, 3)):
        out = tt.full((12, 4, D), 7.0, dtype=tt.float16, device="cuda")
        lay.paged_attention(4, 2, causal=causal)(q, kp, vp, table, ints(lens), ints([0, 2, 5, 10]), out=out)
        assert (out[10:] == 7).all() and (out[2:5] == 0).all()
        if lens[0] <= 0:
            assert (out[:2] == 0).all()
        empty = (out[5:10].reshape(5, -1) == 0).all(-1).tolist()
        # five new rows of a sequence that holds three tokens: the first two see nothing
        assert empty == ([lens[2] == 0] * 5 if not causal or lens[2] == 0 else [True, True, False, False, False])
    # sequences whose rows lie outside of q have none
    out = tt.full((12, 4, D), 7.0, dtype=tt.float16, device="cuda")
    lay.paged_attention(4, 2, causal=causal)(q, kp, vp, table, ints((130, 0, 3)), ints([0, 2, 99, 103]), out=out)
    assert (out[2:] == 7).all() and not (out[:2] == 7).any()
    # no pages at all
    none = lay.new_pages(0, 2)
    assert (lay.paged_attention(4, 2)(q, *none, ints([[0]]), ints([12]), ints([0, 12])) == 0).all()
    assert lay.paged_attention(4, 2)(q[:0], kp, vp, table[:0], ints([]), ints([0])).shape == (0, 4, D)


def test_lengths_are_cut_to_the_table_and_to_max_context():
    lay = layer("turbo4", "turbo4")
    kp, vp, table = filled(lay, (256, 256), 2, 20)
    q = tt.randn((2, 4, D), device="cuda").half()
    attn = lay.paged_attention(4, 2)
    assert tt.equal(attn(q, kp, vp, table, ints([2 ** 31 - 1, 300])), attn(q, kp, vp, table, ints([256, 256])))
    assert tt.equal(attn(q, kp, vp, table, ints([256, 50]), max_context=100), attn(q, kp, vp, table, ints([100, 50]), max_context=100))


def test_rows_from_max_new_on_are_left_as_they_were():
    lay = layer("turbo3", "turbo2")
    lens, new = (400, 300, 50), (40, 3, 20)
    kp, vp, table = filled(lay, lens, 2, 23)
    q = tt.randn((63, 4, D), device="cuda").half()
    attn = lay.paged_attention(4, 2)
    whole = attn(q, kp, vp, table, ints(lens), cumulative(new), max_new=40)
    out = tt.full_like(q, 7.0)
    attn(q, kp, vp, table, ints(lens), cumulative(new), max_new=2, out=out)
    for lo, hi in ((0, 2), (40, 42), (43, 45)):
        assert (out[lo:hi].float() - whole[lo:hi].float()).abs().max() < 2e-3 * 4    # another order of the sums, values of N(0, 1)
        out[lo:hi] = 7
    assert (out == 7).all()


def test_strided_queries_and_tables_and_a_shared_page():
    lay, lens, new = layer("turbo3", "turbo3"), (300, 200, 129), (9, 1, 20)
    kp, vp, table = filled(lay, lens, 2, 21)
    table[1, 0] = table[0, 0]       # a prefix that two sequences share
    q = tt.randn((30, 8, D), device="cuda").bfloat16()
    want, tol = attend64(lay, q, kp, vp, table, lens, new, True)
    attn = lay.paged_attention(8, 2)
    got = attn(q, kp, vp, table, ints(lens), cumulative(new))
    check(got, want, tol)
    wide = tt.full((3, 9), -7, dtype=tt.int32, device="cuda")
    wide[:, :3] = table
    for x in (tt.cat([q, q], 1)[:, :8], tt.cat([q, q], 2)[..., :D], q.transpose(0, 1).contiguous().transpose(0, 1),
              tt.cat([q.flatten(1), q[:, 0, :3]], 1)[:, :8 * D].unflatten(1, (8, D))):
        assert not x.is_contiguous() and tt.equal(attn(x, kp, vp, wide[:, :3], ints(lens), cumulative(new)), got)


def test_results_do_not_depend_on_the_neighbours_and_repeat():
    """The same sequence alone and in a batch of a hundred (two rounds of the batch's look-up), twice."""
    lay = layer("turbo3", "turbo4")
    lens = [(53 * b) % 400 + 1 for b in range(100)]
    new = [(b % 3) * (b % 2) * 4 % (c + 1) for b, c in enumerate(lens)]
    kp, vp, table = filled(lay, lens, 1, 22)
    q = tt.randn((sum(new), 4, D), device="cuda").half()
    attn = lay.paged_attention(4, 1)
    got = attn(q, kp, vp, table, ints(lens), cumulative(new))
    assert tt.equal(got, attn(q, kp, vp, table, ints(lens), cumulative(new)))
    want, tol = attend64(lay, q, kp, vp, table, lens, new, True)
    check(got, want, tol)


def test_pools_beyond_32_bits():
    """A pool of 5 GB per side, the sequence's pages at its far end."""
    lay, hkv = layer("q8_0", "q8_0"), 8
    n = 5 * 2 ** 30 // (hkv * 128 * 136)
    kp, vp = lay.new_pages(n, hkv)
    small = lay.new_pages(3, hkv)
    table = ints([[n - 1, n - 3, n - 2]])
    near = ints([[2, 0, 1]])
    k, v, q = (tt.randn((300, h, D), device="cuda").half() for h in (hkv, hkv, 16))
    lay.append_paged(k, v, kp, vp, table, ints([0]), cumulative([300]))
    lay.append_paged(k, v, *small, near, ints([0]), cumulative([300]))
    assert tt.equal(kp[-3:], small[0]) and tt.equal(vp[-3:], small[1]) and not kp[:-3].any()
    attn = lay.paged_attention(16, hkv)
    assert tt.equal(attn(q, kp, vp, table, ints([300]), cumulative([300])), attn(q, *small, near, ints([300]), cumulative([300])))
    assert all(tt.equal(a, b) for a, b in zip(lay.load_paged(kp, vp, table, ints([0]), cumulative([300]), 300),
                                              lay.load_paged(*small, near, ints([0]), cumulative([300]), 300)))


@pytest.mark.parametrize("kf,vf", [("q8_0", "turbo4"), ("turbo4", "turbo4")])
def test_few_rows_in_pools_beyond_32_bits(kf, vf):
    """The other kernels: single tokens with and without 4-bit tables of a copy per lane, 16, 24, 48 and 60 rows."""
    lay, hkv, c = layer(kf, vf), 8, 3000
    n = int(4.5 * 2 ** 30) // (hkv * 128 * 66)
    kp, vp = lay.new_pages(n, hkv)
    blocks = -(-c // 128)
    small = lay.new_pages(blocks, hkv)
    table, near = ints([[n - 1 - i for i in range(blocks)]]), ints([list(range(blocks))])
    k, v = (tt.randn((c, hkv, D), device="cuda").half() for _ in range(2))
    lay.append_paged(k, v, kp, vp, table, ints([0]), cumulative([c]))
    lay.append_paged(k, v, *small, near, ints([0]), cumulative([c]))
    attn = lay.paged_attention(16, hkv)
    for new in (1, 8, 12, 24, 30):
        q = tt.randn((new, 16, D), device="cuda").half()
        assert tt.equal(attn(q, kp, vp, table, ints([c]), cumulative([new])), attn(q, *small, near, ints([c]), cumulative([new]))), new
    many = 32
    q = tt.randn((many, 16, D), device="cuda").half()      # a prefix that all of a batch share
    got, want = (attn(q, *pools, rows.expand(many, blocks).contiguous(), ints([c] * many)) for pools, rows in (((kp, vp), table), (small, near)))
    assert tt.equal(got, want)


# ---- a serving loop --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kf,vf", [("turbo3", "turbo3"), ("q8_0", "turbo4")])
def test_serving_loop(kf, vf):
    """Prompts in two chunks, drafted tokens, single steps of two users, rotary positions first: every step against 64 bits on
    the pages and the steps of one token against the contiguous cache's attention."""
    lay, hq, hkv = layer(kf, vf), 8, 2
    rot = tqa.Rotary(D, base=500000.0)
    kp, vp = lay.new_pages(9, hkv)
    table = ints([[8, 2, 5, 0], [1, 7, 3, 6]])
    cap = 512
    whole = [lay.new_cache(hkv, cap) for _ in range(2)]
    lens = np.array([0, 0])
    gen = tt.Generator("cuda").manual_seed(30)
    attn = lay.paged_attention(hq, hkv)
    for new in ([130, 7], [60, 250], [4, 4], [1, 1], [1, 1]):
        qkv = tt.randn((sum(new), (hq + 2 * hkv) * D), generator=gen, device="cuda").half()
        q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([hq * D, hkv * D, hkv * D], 1))
        pos = tt.cat([tt.arange(int(c), int(c) + n, device="cuda") for c, n in zip(lens, new)])
        rot(q, k, pos, out=(q, k))
        lay.append_paged(k, v, kp, vp, table, ints(lens.tolist()), cumulative(new))
        at = 0
        for b, n in enumerate(new):
            lay.append(*(x[at:at + n].transpose(0, 1).contiguous() for x in (k, v)), *whole[b], int(lens[b]), cap)
            at += n
        lens += new
        got = attn(q, kp, vp, table, ints(lens.tolist()), None if new == [1, 1] else cumulative(new), max_context=512)
        want, tol = attend64(lay, q, kp, vp, table, lens.tolist(), new, True)
        check(got, want, tol)
        if new == [1, 1]:
            for b in range(2):
                one = lay.attention(1, hq, hkv, int(lens[b]), capacity=cap)(q[b:b + 1].contiguous(), *whole[b])
                assert (one[0] - got[b].float()).abs().max() < 4e-3 * one.abs().max()     # that one's own 2e-3, twice


def test_captured_step_replays_while_the_cache_grows():
    lay, hq, hkv = layer("turbo3", "turbo4"), 8, 2
    rot, attn = tqa.Rotary(D), lay.paged_attention(8, 2)
    kp, vp, table = filled(lay, (250, 3), hkv, 31, extra=4, width=4)
    for b in range(2):
        spare = [p for p in range(kp.shape[0]) if p not in table.flatten().tolist()]
        for i in range(4):
            if table[b, i] < 0 and spare:
                table[b, i] = spare.pop()
    k2, v2 = kp.clone(), vp.clone()
    lens, word = ints([250, 3]), tt.zeros(1, dtype=tt.int32, device="cuda")
    q, k, v = (tt.zeros((2, h, D), device="cuda", dtype=tt.float16) for h in (hq, hkv, hkv))
    out = tt.empty_like(q)

    def step(kp, vp, out):
        turned = rot(q, k, lens)
        lay.append_paged(turned[1], v, kp, vp, table, lens, overrun=word)
        lens.add_(1)
        return attn(turned[0], kp, vp, table, lens, out=out)

    side = tt.cuda.Stream()
    side.wait_stream(tt.cuda.current_stream())
    with tt.cuda.stream(side):
        step(kp, vp, out)
    tt.cuda.current_stream().wait_stream(side)
    lens.sub_(1)
    graph = tt.cuda.CUDAGraph()
    with tt.cuda.graph(graph):
        step(kp, vp, out)
    kp.copy_(k2), vp.copy_(v2)
    gen = tt.Generator("cuda").manual_seed(32)
    for i in range(12):         # over the block's end
        for x in (q, k, v):
            x.copy_(tt.randn(x.shape, generator=gen, device="cuda"))
        before = lens.clone()
        graph.replay()
        tt.cuda.synchronize()
        got, after = out.clone(), lens.clone()
        lens.copy_(before)
        want = step(k2, v2, tt.empty_like(out))
        assert tt.equal(after, lens) and tt.equal(kp, k2) and tt.equal(vp, v2) and tt.equal(got, want), i
    assert overrun_bits(word) == 0


def test_another_stream():
    lay, lens = layer("turbo3", "turbo3"), (900, 40)
    kp, vp, table = filled(lay, lens, 2, 33)
    q = tt.randn((2, 8, D), device="cuda").half()
    attn = lay.paged_attention(8, 2)
    want = attn(q, kp, vp, table, ints(lens))
    args = ints(lens)
    side = tt.cuda.Stream()
    side.wait_stream(tt.cuda.current_stream())
    with tt.cuda.stream(side):
        got = attn(q, kp, vp, table, args)
    side.synchronize()
    assert tt.equal(got, want)


def test_refusals():
    lay = layer("turbo3", "q8_0")
    kp, vp = lay.new_pages(4, 2)
    table, lens, cu = ints([[0, 1], [2, 3]]), ints([5, 6]), ints([0, 3, 6])
    k = tt.zeros((6, 2, D), device="cuda", dtype=tt.float16)
    q = tt.zeros((6, 4, D), device="cuda", dtype=tt.float16)
    attn = lay.paged_attention(4, 2)
    app = lambda k=k, v=k, kp=kp, vp=vp, table=table, lens=lens, cu=cu, **kw: lay.append_paged(k, v, kp, vp, table, lens, cu, **kw)
    att = lambda q=q, kp=kp, vp=vp, table=table, lens=lens, cu=cu, **kw: attn(q, kp, vp, table, lens, cu, **kw)
    for call, error, text in [
            (lambda: app(k=k[:5]), ValueError, "same rows"), (lambda: app(v=k.float()), ValueError, "same rows"),
            (lambda: app(k=k.double(), v=k.double()), TypeError, "float64"), (lambda: app(k=k[:, :1]), ValueError, r"must be \[rows, 2"),
            (lambda: app(k=k.cpu()), ValueError, "current device"), (lambda: app(kp=kp.cpu()), ValueError, "current device"),
            (lambda: app(kp=vp, vp=kp), ValueError, "k_pages must be"), (lambda: app(kp=kp[:3]), ValueError, "same pages"),
            (lambda: app(kp=kp[:, :1]), ValueError, "k_pages must be"), (lambda: app(table=table.long()), ValueError, "block_table"),
            (lambda: app(table=table.t()), ValueError, "block_table"), (lambda: app(table=table.cpu()), ValueError, "current device"),
            (lambda: app(lens=lens[:1]), ValueError, "lengths"), (lambda: app(lens=lens.long()), ValueError, "lengths"),
            (lambda: app(cu=cu[:2]), ValueError, "cu_new"), (lambda: app(cu=cu.cpu()), ValueError, "current device"),
            (lambda: app(overrun=lens), ValueError, "overrun"), (lambda: app(k=k[:1], v=k[:1], cu=None), ValueError, "1 rows for 2"),
            (lambda: lay.load_paged(kp, vp, table, lens, cu), ValueError, "number of rows"),
            (lambda: lay.load_paged(kp, vp, table, lens, cu, out=(k, k.float())), ValueError, "outputs"),
            (lambda: att(q=q.float()), TypeError, "float32"), (lambda: att(q=q[:, :3]), ValueError, r"must be \[rows, 4"),
            (lambda: att(out=q[:5]), ValueError, "out must"), (lambda: att(out=q.bfloat16()), ValueError, "out must"),
            (lambda: att(q=q.cpu()), ValueError, "current device"), (lambda: att(max_context=-1), ValueError, "negative"),
            (lambda: lay.paged_attention(4, 4)(q, kp, vp, table, lens, cu), ValueError, "KV heads"),
            (lambda: lay.paged_attention(4, 2, scale=0.0)(q, kp, vp, table, lens, cu), ValueError, "scale")]:
        with pytest.raises(error, match=text):
            call()
