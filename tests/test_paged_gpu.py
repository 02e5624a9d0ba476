"""s2t_amd.paged (csrc/paged.hip): the paged key/value cache and attention of several new tokens over it, against the definitions in float64
on the CPU.

Bounds of the attention.  e = 2^-24.  A score is a sum of d products of exactly held factors times scale * log2(e): within
ES = e (d + 4) * max over keys of scale * sum |q k|.  exp then has that as a relative error, with the rounding of its argument (below
the largest |score| difference, itself below 2 max |score| <= 2 ES / (e (d + 4))) and 2 steps of the hardware's.  Probabilities may be held
as two bf16 numbers, 2^-16 of the value.  A sum over n keys in blocks costs at most n e, the final rounding half a step (2^-8 of the value
in bf16).  With A = sum p |v|: |out - exact| <= half |exact| + A (2 (2 ES) + 2^-16 + 2^-21 + 2 (n + 64) e), the factor 2 because numerator and
denominator both move.  lse moves by 2 ES + (n + 64) e + 2^-21 + 2 e |lse|.
Those of the append: a copy is exact; a rotated element is two products and a sum in fp32 (3 e of |x| + |y|) and one rounding."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from s2t_amd import modules  # noqa: E402
from s2t_amd import paged  # noqa: E402

DEV = "cuda"
E = 2.0 ** -24
HALF = {torch.float32: E, torch.bfloat16: 2.0 ** -8}


def make(news, ctxs, Hq, Hkv, d, page, dtype, seed, spare=3, order="phsd", garbage=None):
    """A cache with scattered pages; places behind a sequence's end hold ``garbage`` where given."""
    r = np.random.RandomState(seed)
    g = torch.Generator().manual_seed(seed)
    B = len(news)
    lens = np.array(news) + np.array(ctxs)
    used = -(-lens // page)
    P = int(used.sum()) + spare
    table = np.full((B, max(1, int(used.max()))), -1, dtype=np.int32)
    perm, at = r.permutation(P), 0
    for b, u in enumerate(used):
        table[b, :u] = perm[at:at + u]
        at += u
    shape = (P, Hkv, page, d) if order == "phsd" else (P, page, Hkv, d)
    k, v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    if order != "phsd":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    if garbage is not None:
        keep = torch.zeros(P, page, dtype=torch.bool)
        for b in range(B):
            for p in range(int(lens[b])):
                keep[table[b, p // page], p % page] = True
        for x in (k, v):
            x.transpose(1, 2)[~keep] = garbage
    N = int(sum(news))
    c = dict(B=B, N=N, news=list(news), lens=lens, table=table, k=k, v=v, page=page, d=d, Hq=Hq, Hkv=Hkv, dtype=dtype,
             cu=np.concatenate([[0], np.cumsum(news)]).astype(np.int32), q=torch.randn(N, Hq, d, generator=g).to(dtype), g=g, r=r)
    return c


def on_gpu(c, extra_rows=0):
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(DEV)  # noqa: E731
    q = torch.cat([c["q"], torch.full((extra_rows, c["Hq"], c["d"]), math.nan, dtype=c["dtype"])]) if extra_rows else c["q"]
    return dict(q=q.to(DEV), k_pages=c["k"].to(DEV), v_pages=c["v"].to(DEV), page_table=dev(c["table"]), lens=dev(c["lens"].astype(np.int32)),
                cu=dev(c["cu"]), max_new=max(c["news"] + [0]))


def random_tree(c, words=None, empty=()):
    """Ancestors and itself, the parent any earlier node or the prefix; rows in ``empty`` see no new token."""
    W = words or max(1, -(-max(c["news"]) // 64))
    sees = np.zeros((c["N"], 64 * W), dtype=bool)
    for b, n in enumerate(c["news"]):
        for i in range(n):
            t = c["cu"][b] + i
            p = c["r"].randint(-1, i) if i else -1
            if p >= 0:
                sees[t] = sees[c["cu"][b] + p]
            sees[t, i] = True
    for t in empty:
        sees[t] = False
    return sees, torch.from_numpy(np.packbits(sees, axis=1, bitorder="little").view(np.int64).copy())


def exact(c, sees=None, scale=None, visible=None):
    """-> out, lse, bound of out, bound of lse (float64).  ``visible(b, place)``: further keys that do not exist."""
    scale = c["d"] ** -0.5 if scale is None else scale
    G = c["Hq"] // c["Hkv"]
    out = torch.zeros(c["N"], c["Hq"], c["d"], dtype=torch.float64)
    lse = torch.full((c["N"], c["Hq"]), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for b, n in enumerate(c["news"]):
        L = int(c["lens"][b])
        if n == 0 or L == 0:
            continue
        place = np.arange(L)
        page = torch.from_numpy(c["table"][b][place // c["page"]].astype(np.int64))
        ok = np.ones(L, dtype=bool) if visible is None else np.array([visible(b, p) for p in place])
        k = c["k"][page.clamp(0, c["k"].shape[0] - 1), :, torch.from_numpy(place % c["page"])].double().transpose(0, 1).repeat_interleave(G, 0)
        v = c["v"][page.clamp(0, c["k"].shape[0] - 1), :, torch.from_numpy(place % c["page"])].double().transpose(0, 1).repeat_interleave(G, 0)
        q = c["q"][c["cu"][b]:c["cu"][b + 1]].double().transpose(0, 1)
        j = place - (L - n)
        m = np.zeros((n, L), dtype=bool)
        for i in range(n):
            m[i] = (j < 0) | ((j <= i) if sees is None else sees[c["cu"][b] + i][np.clip(j, 0, sees.shape[1] - 1)] & (j < sees.shape[1]))
        m &= ok[None]
        mask = torch.from_numpy(m)
        for i in range(n):
            cols = mask[i].nonzero().flatten()
            if not len(cols):
                continue
            t = c["cu"][b] + i
            s = (k[:, cols] @ q[:, i, :, None])[..., 0] * scale
            es = E * (c["d"] + 4) * ((k[:, cols].abs() @ q[:, i, :, None].abs())[..., 0] * abs(scale)).amax(1)
            es = es + 2 * E * s.abs().amax(1)
            p = torch.softmax(s, -1)
            out[t] = (p[:, None] @ v[:, cols])[:, 0]
            lse[t] = torch.logsumexp(s, -1)
            A = (p[:, None] @ v[:, cols].abs())[:, 0]
            tol[t] = HALF[c["dtype"]] * out[t].abs() + A * (4 * es + 2.0 ** -16 + 2.0 ** -21 + 2 * (len(cols) + 64) * E)[:, None] + 1e-37
            ltol[t] = 2 * es + (len(cols) + 64) * E + 2.0 ** -21 + 2 * E * lse[t].abs()
    return out, lse, tol, ltol


def check(c, got, sees=None, scale=None, visible=None):
    out, lse, tol, ltol = exact(c, sees, scale, visible)
    o, l = got[0][:c["N"]].cpu().double(), got[1][:c["N"]].cpu().double()
    none = torch.isinf(lse)
    assert torch.equal(torch.isinf(l), none) and not o[none].any()
    worst = ((o - out).abs() / tol.clamp(min=1e-300))[~none]
    assert bool(((o - out).abs() <= tol).all()), (float(worst.max()) if worst.numel() else 0.0, int(((o - out).abs() > tol).sum()))
    assert bool(((l - lse).abs() <= ltol)[~none].all()), float((l - lse)[~none].abs().max())


# (new tokens, cache in front of them) of each sequence, query heads, key/value heads, head_dim, page_size
SHAPES = [
    ([1], [0], 1, 1, 16, 16),
    ([1], [1], 1, 1, 64, 1),
    ([1, 1, 1], [0, 5, 300], 4, 4, 64, 16),
    ([1] * 5, [15, 16, 17, 31, 1000], 8, 2, 64, 32),
    ([1, 0, 3, 0], [40, 7, 0, 0], 2, 2, 32, 8),
    ([5, 13, 1, 2], [63, 64, 65, 127], 6, 2, 48, 16),
    ([33, 17], [100, 1], 3, 1, 80, 64),
    ([70, 130, 64], [10, 0, 250], 4, 4, 64, 64),
    ([9, 2], [500, 33], 4, 1, 128, 256),
    ([7, 20], [90, 3], 2, 1, 256, 4),
    ([2], [5000], 16, 2, 64, 128),
    ([257], [300], 2, 2, 112, 2),
    ([17, 30, 1, 0] * 16, [0, 90, 40, 7] * 16, 8, 4, 64, 16),      # few keys, many rows: waves with rows of their own
    ([5, 40] * 24, [100, 3] * 24, 12, 6, 32, 4),
    ([23] * 66, [9] * 66, 4, 4, 128, 32),
]


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_against_float64(shape, dtype, tree):
    c = make(*shape, dtype=dtype, seed=len(shape[0]) * 100 + shape[4])
    sees, words = random_tree(c) if tree else (None, None)
    check(c, paged.paged_attention(**on_gpu(c), tree=words.to(DEV) if tree else None, return_lse=True), sees)


# keys in ranges (one workgroup each, joined afterwards): two ranges of 128 keys, ranges that end inside the new tokens, sequences with one range
# next to some with several, up to 256 of them
RANGES = [
    ([1, 1], [255, 254], 1, 1, 256, 16),
    ([1, 7, 2], [383, 129, 3], 2, 2, 128, 16),
    ([40, 1, 0, 3], [230, 600, 500, 90], 2, 1, 256, 32),
    ([3, 64], [2100, 450], 4, 1, 64, 1),
    ([2, 1], [40000, 9], 2, 2, 16, 64),
    ([1], [133000], 1, 1, 64, 256),
    ([5], [33000], 4, 1, 128, 128),
]


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", RANGES)
def test_keys_in_ranges(shape, dtype, tree):
    c = make(*shape, dtype=dtype, seed=500 + shape[4])
    sees, words = random_tree(c) if tree else (None, None)
    check(c, paged.paged_attention(**on_gpu(c), tree=words.to(DEV) if tree else None, return_lse=True), sees)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_see_nothing(dtype):
    """No prefix and no bits; a whole sequence of such rows next to ordinary ones; a prefix but no bits is an ordinary row."""
    c = make([3, 20, 2, 18], [0, 0, 7, 0], 4, 2, 64, 16, dtype, 5)
    sees, words = random_tree(c, empty=[0, 2, 5, 6, 23, 24] + list(range(25, 43)))
    check(c, paged.paged_attention(**on_gpu(c), tree=words.to(DEV), return_lse=True), sees)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mask_words_bits_behind_the_new_tokens_and_too_few_words(dtype):
    """Set bits behind a sequence's new tokens mean nothing; new tokens behind the last word are not seen; any set of bits will do (bit 63,
    later tokens, not itself)."""
    c = make([70, 3, 64], [5, 40, 0], 2, 2, 64, 16, dtype, 6)
    sees = c["r"].rand(c["N"], 128) < 0.4
    pack = lambda s: torch.from_numpy(np.packbits(s, axis=1, bitorder="little").view(np.int64).copy()).to(DEV)  # noqa: E731
    check(c, paged.paged_attention(**on_gpu(c), tree=pack(sees), return_lse=True), sees)
    check(c, paged.paged_attention(**on_gpu(c), tree=pack(sees)[:, :1], return_lse=True), sees[:, :64])


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_a_row_does_not_see_never_touches_it(dtype, value):
    """Free pages, places behind a sequence's end, and new tokens that the tree hides hold NaN or infinities in keys and values."""
    c = make([6, 1, 40, 20], [30, 0, 77, 0], 4, 2, 64, 16, dtype, 7, garbage=value)
    sees, words = random_tree(c)
    check(c, paged.paged_attention(**on_gpu(c), tree=words.to(DEV), return_lse=True), sees)
    check(c, paged.paged_attention(**on_gpu(c), return_lse=True))
    # new tokens 2 and 5 of sequence 0, 39 of sequence 2, 0 of sequence 3: hidden from the others by the tree, and poisoned
    poisoned = [(0, 2), (0, 5), (2, 39), (3, 0)]
    clean = {x: c[x].clone() for x in "kv"}
    for b, j in poisoned:
        sees[c["cu"][b]:c["cu"][b + 1], j] = False
        place = int(c["lens"][b]) - c["news"][b] + j
        for x in "kv":
            c[x][c["table"][b, place // 16], :, place % 16] = value
    words = torch.from_numpy(np.packbits(sees, axis=1, bitorder="little").view(np.int64).copy())
    got = paged.paged_attention(**on_gpu(c), tree=words.to(DEV), return_lse=True)
    c.update(clean)
    check(c, got, sees)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_values_that_are_seen(dtype):
    """An infinity in a value reaches the rows that see it, in its column, and no other; one row of values with a NaN likewise."""
    c = make([6, 3], [20, 4], 2, 2, 64, 16, dtype, 8)
    sees, words = random_tree(c)
    b, j, place = 0, 3, 23
    c["v"][c["table"][b, place // 16], 0, place % 16, 17] = math.inf
    c["v"][c["table"][b, place // 16], 0, place % 16, 40] = math.nan
    c["v"][c["table"][1, 0], 1, 2, 5] = -math.inf  # in the prefix: all rows of sequence 1
    out, _ = paged.paged_attention(**on_gpu(c), tree=words.to(DEV), return_lse=True)
    out = out.cpu().float()
    for t in range(9):
        inf, nan = out[t].isinf().nonzero().tolist(), out[t].isnan().nonzero().tolist()
        if t < 6:
            assert inf == ([[0, 17]] if sees[t, j] else []) and nan == ([[0, 40]] if sees[t, j] else [])
        else:
            assert inf == [[1, 5]] and nan == []


@pytest.mark.parametrize("splits", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nan_scores_that_are_seen(dtype, splits):
    """A NaN in a key makes the rows that see it NaN (those that see nothing else too), and no other row; so does one in a query."""
    c = make([6, 1, 2], [20 if not splits else 3000, 0, 40], 2, 2, 64, 16, dtype, 12)
    sees, words = random_tree(c)
    place = int(c["lens"][0]) - 6 + 3                                              # new token 3 of sequence 0, head 1
    c["k"][c["table"][0, place // 16], 1, place % 16, 5] = math.nan
    c["k"][c["table"][1, 0], 0, 0, 0] = math.nan                                   # all that sequence 1's only token sees in head 0
    c["q"][8, 1, 2] = math.nan
    out, lse = (x.cpu().float() for x in paged.paged_attention(**on_gpu(c), tree=words.to(DEV), return_lse=True))
    want = torch.zeros(9, 2, dtype=torch.bool)
    want[:6, 1] = torch.from_numpy(sees[:6, 3])
    want[6, 0] = want[8, 1] = True
    assert torch.equal(lse.isnan(), want) and torch.equal(out.isnan(), want[..., None].expand(9, 2, 64))
    assert out[~want].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_scores_and_a_scale_of_ones_own(dtype):
    """Scores of several hundred: the running maximum has to carry the sum; a negative and a zero scale are scales too."""
    c = make([5, 2], [300, 64], 2, 1, 64, 16, dtype, 9)
    c["q"] = c["q"] * 8
    for scale in (2.0, -0.3, 0.0):
        check(c, paged.paged_attention(**on_gpu(c), scale=scale, return_lse=True), scale=scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ctx", [20, 250, 1500, 40000])
@pytest.mark.parametrize("power", [4, 14, 22, 31, 40, 90, 120])
@pytest.mark.parametrize("sign", [1, -1])
def test_equal_scores_of_any_size_share_the_weight(sign, power, ctx, dtype):
    """Scores are powers of two or their double (of the other sign's: half), exact in every type: the keys of the largest score share the
    weight to the rounding of one sum, whatever its size, and wherever among the others they stand.  out = mean of their values, within
    A (2^-16 + 2^-21 + 2 (n + 64) e) and the rounding of the result; lse = score + log n within 2 e of its size and 2^-20."""
    d = 64
    c = make([3], [ctx], 2, 1, d, 16, dtype, seed=power + ctx)
    c["q"].zero_()
    c["q"][:, :, 5] = 2.0
    c["k"].zero_()
    low, high = sorted((sign * 2.0 ** power, sign * 2.0 ** (power + 1)))
    L = ctx + 3
    place = np.arange(L)
    tops = torch.from_numpy(c["r"].rand(L) < 0.3)
    tops[0] = True
    page, slot = torch.from_numpy(c["table"][0][place // 16].astype(np.int64)), torch.from_numpy(place % 16)
    c["k"][page, :, slot, 5] = torch.where(tops, torch.tensor(high), torch.tensor(low)).to(dtype)[:, None]
    out, lse = paged.paged_attention(**on_gpu(c), scale=0.25, return_lse=True)
    v = c["v"][page, 0, slot].double()
    for i in range(3):
        s = torch.where(tops, high / 2, low / 2)[:ctx + i + 1].double()
        p = torch.softmax(s, 0)
        want, A = p @ v[:ctx + i + 1], p @ v[:ctx + i + 1].abs()
        es = 2 * E * 4 if power > 10 else 16 * E * 2.0 ** power  # (differences are either 0 or so large that the other side is 0)
        tol = HALF[dtype] * want.abs() + A * (4 * es + 2.0 ** -16 + 2.0 ** -21 + 2 * (L + 64) * E) + 1e-37
        l = float(torch.logsumexp(s, 0))
        for hq in range(2):
            assert bool(((out[i, hq].cpu().double() - want).abs() <= tol).all()), float(((out[i, hq].cpu().double() - want).abs() / tol).max())
            assert abs(float(lse[i, hq]) - l) <= 4 * E * abs(l) + (L + 64) * E + 2.0 ** -20


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_strides_and_rows_behind_the_last_sequence(dtype):
    """Pages as a view of [pages, page, heads, d], queries and outputs inside wider rows, a table inside a wider one, a loose max_new; rows
    behind the last sequence are left as they were."""
    c = make([4, 0, 19], [50, 9, 200], 4, 2, 64, 32, dtype, 10, order="pshd")
    a = on_gpu(c, extra_rows=5)
    assert not a["k_pages"].is_contiguous()
    wide = torch.zeros(c["N"] + 5, 10, 64, dtype=dtype, device=DEV)
    wide[:, 3:7] = a["q"]
    a["q"] = wide[:, 3:7]
    table = torch.full((3, 40), 1 << 30, dtype=torch.int32, device=DEV)
    table[:, :a["page_table"].shape[1]] = a["page_table"]
    a["page_table"] = table[:, :a["page_table"].shape[1]]
    a["max_new"] = 40
    o = torch.full((c["N"] + 5, 8, 64), 7.0, dtype=dtype, device=DEV)
    got = paged.paged_attention(**a, out=o[:, 2:6], return_lse=True)
    check(c, got)
    assert bool((o[:, :2] == 7).all()) and bool((o[:, 6:] == 7).all()) and bool((o[c["N"]:] == 7).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_entries_that_lead_out_of_bounds_are_never_followed(dtype):
    """Pages that do not exist (negative, too large), a length beyond the table, fewer places than new tokens, a cu that runs backwards or
    beyond the rows: such keys do not exist, such rows are not computed, everything else comes out as ever."""
    c = make([3, 2, 4, 3], [60, 100, 10, 0], 4, 2, 64, 16, dtype, 11)
    c["table"][0, 1], c["table"][1, 3] = -5, 1 << 30
    a = on_gpu(c)
    check(c, paged.paged_attention(**a, return_lse=True), visible=lambda b, p: not (b == 0 and 16 <= p < 32 or b == 1 and 48 <= p < 64))
    # sequence 2 claims a length beyond its table's row: only what the table holds exists (14 places were meant, 7 * 16 = 112 can exist)
    c2 = make([3, 2, 4, 3], [60, 100, 10, 0], 4, 2, 64, 16, dtype, 11)
    a = on_gpu(c2)
    a["lens"][3] = 2  # three new tokens in two places: the first one's place is -1
    o, l = paged.paged_attention(**a, return_lse=True)
    t = int(c2["cu"][3])
    assert float(l[t].max()) == -math.inf and not o[t].any() and torch.isfinite(l[t + 1:]).all()
    a["lens"][3] = 1 << 30
    o, l = paged.paged_attention(**a, return_lse=True)
    torch.cuda.synchronize()
    a = on_gpu(c2)
    a["cu"] = torch.tensor([0, 3, 1, 900, 2], dtype=torch.int32, device=DEV)
    o = torch.full_like(a["q"], 3.0)
    paged.paged_attention(**a, out=o)
    k, v = (torch.randn(c2["N"], 2, 64, device=DEV).to(dtype) for _ in range(2))
    a.pop("q")
    paged.paged_kv_append(k, v, **a)
    torch.cuda.synchronize()
    assert torch.isfinite(o[:3]).all()


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_length_beyond_the_table_means_all_its_keys(dtype, tree):
    """A sequence that claims 2^30 places sees every key that its table's row holds and nothing else (its new tokens' places are not among
    them, so a tree hides nothing), the others are bit for bit what they are without it."""
    c = make([3, 2, 4, 3], [60, 100, 10, 0], 4, 2, 64, 16, dtype, 11)
    c["table"][3] = np.array([3, -1, 5, 1 << 30, 0, 2, 1])[:c["table"].shape[1]]   # (pages of other sequences will do for keys)
    assert c["table"].shape[1] == 7
    sees, words = random_tree(c) if tree else (None, None)
    more = dict(tree=words.to(DEV) if tree else None, return_lse=True)
    a = on_gpu(c)
    before = paged.paged_attention(**a, **more)
    a["lens"][3] = 1 << 30
    o, l = paged.paged_attention(**a, **more)
    t = int(c["cu"][3])
    assert torch.equal(o[:t], before[0][:t]) and torch.equal(l[:t], before[1][:t])
    # the same keys as the prefix of a sequence whose three new tokens lie behind them and are hidden
    c["lens"] = np.array([63, 102, 14, 112 + 3])
    c["table"] = np.concatenate([c["table"], np.full((4, 1), -1, dtype=np.int32)], 1)
    check(c, (o, l), sees, visible=lambda b, p: not (b == 3 and (p >= 112 or 16 <= p < 32 or 48 <= p < 64)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offsets_that_run_backwards_or_beyond_the_rows(dtype):
    """cu = 0, 3, 1, 900, 2 over 12 rows: sequence 0 has rows 0 - 2; sequence 1 none; sequence 2 rows 1 - 11 (11 of the 899 it claims) of
    which ``max_new`` bounds the first four; sequence 3 none.  Row 0 has one owner and is exact; rows 5 - 11 are nobody's and stay as they
    were; the append changes the places of the owned rows alone.  (Rows 1 - 4 come from one owner or the other.)"""
    c = make([3, 2, 4, 3], [60, 100, 10, 0], 4, 2, 64, 16, dtype, 11)
    a = on_gpu(c)
    assert a["max_new"] == 4
    a["cu"] = torch.tensor([0, 3, 1, 900, 2], dtype=torch.int32, device=DEV)
    o = torch.full_like(a["q"], 3.0)
    _, l = paged.paged_attention(**a, out=o, return_lse=True)
    assert bool((o[5:] == 3).all()) and torch.isfinite(o).all()
    out, lse, tol, ltol = exact(c)
    assert bool(((o[0].cpu().double() - out[0]).abs() <= tol[0]).all()) and bool(((l[0].cpu().double() - lse[0]).abs() <= ltol[0]).all())
    # sequence 2: 14 places and 11 rows, the prefix is three places, row 1 + i sees places 0 .. 3 + i; row 3 and 4 are its own alone
    one = dict(c, B=1, N=4, news=[4], lens=np.array([7]), table=c["table"][2:3], cu=np.array([0, 4]), q=c["q"][1:5])
    out, lse, tol, ltol = exact(one)
    assert bool(((o[3:5].cpu().double() - out[2:]).abs() <= tol[2:]).all()) and bool(((l[3:5].cpu().double() - lse[2:]).abs() <= ltol[2:]).all())
    k, v = (torch.randn(c["N"], 2, 64, generator=c["g"]).to(dtype) for _ in range(2))
    want = {x: c[x].clone() for x in "kv"}
    for b, row0, n, place in ((0, 0, 3, 60), (2, 1, 4, 3)):
        for i in range(n):
            for x, src in (("k", k), ("v", v)):
                want[x][c["table"][b, (place + i) // 16], :, (place + i) % 16] = src[row0 + i]
    a.pop("q")
    paged.paged_kv_append(k.to(DEV), v.to(DEV), **a)
    assert torch.equal(a["k_pages"].cpu(), want["k"]) and torch.equal(a["v_pages"].cpu(), want["v"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,rot,page", [(64, 64, 16), (16, 16, 1), (48, 32, 8), (128, 128, 64), (256, 64, 2), (80, 80, 32)])
@pytest.mark.parametrize("select", [False, True])
def test_append_against_float64(dtype, d, rot, page, select):
    news, Hq, Hkv = [1, 0, 7, 40, 3], 6, 2
    c = make(news, [0, 5, 15, 16, 90], Hq, Hkv, d, page, dtype, d + page)
    N = c["N"]
    src = N + 9 if select else N
    fused = torch.randn(src, Hq + 2 * Hkv, d, generator=c["g"]).to(dtype)
    rows = torch.from_numpy(c["r"].permutation(src)[:N].astype(np.int32)) if select else None
    tab = modules.rotary_table(200, rot)
    pos = torch.from_numpy(c["r"].randint(0, 200, N).astype(np.int32))
    f = fused.to(DEV)
    for rotary, positions in ((None, None), (tab, None), (tab, pos)):
        a = on_gpu(c)
        a.pop("q")
        q = None if select else f[:, :Hq]
        got_q = paged.paged_kv_append(f[:, Hq:Hq + Hkv], f[:, Hq + Hkv:], **a, q=q, rotary=rotary.to(DEV) if rotary is not None else None,
                                      positions=positions.to(DEV) if positions is not None else None, rows=rows.to(DEV) if select else None)
        want = {x: c[x].clone() for x in "kv"}
        for b, n in enumerate(news):
            for i in range(n):
                t, place = int(c["cu"][b]) + i, int(c["lens"][b]) - n + i
                row = fused[int(rows[t]) if select else t].double()
                p = place if positions is None else int(positions[t])

                def turned(x):
                    if rotary is None:
                        return x, torch.zeros_like(x)
                    y, w = x.clone(), torch.zeros_like(x)
                    cs, sn = rotary[p, :rot // 2].double(), rotary[p, rot // 2:].double()
                    x1, x2 = x[:, :rot // 2], x[:, rot // 2:rot]
                    y[:, :rot // 2], y[:, rot // 2:rot] = x1 * cs - x2 * sn, x2 * cs + x1 * sn
                    w[:, :rot] = HALF[dtype] * y[:, :rot].abs() + 3 * E * (x1.abs() + x2.abs()).repeat(1, 2) + 1e-38
                    return y, w

                page_, slot = c["table"][b, place // page], place % page
                y, w = turned(row[Hq:Hq + Hkv])
                assert bool(((a["k_pages"][page_, :, slot].cpu().double() - y).abs() <= w).all())
                assert torch.equal(a["v_pages"][page_, :, slot].cpu().double(), row[Hq + Hkv:])
                want["k"][page_, :, slot], want["v"][page_, :, slot] = a["k_pages"][page_, :, slot].cpu(), a["v_pages"][page_, :, slot].cpu()
                if not select:
                    y, w = turned(row[:Hq])
                    assert bool(((got_q[t].cpu().double() - y).abs() <= w).all())
        assert torch.equal(a["k_pages"].cpu(), want["k"]) and torch.equal(a["v_pages"].cpu(), want["v"])  # nothing else was touched
        if not select:  # in place
            again = f.clone()
            a2 = on_gpu(c)
            a2.pop("q")
            r = paged.paged_kv_append(again[:, Hq:Hq + Hkv], again[:, Hq + Hkv:], **a2, q=again[:, :Hq], q_out=again[:, :Hq],
                                      rotary=rotary.to(DEV) if rotary is not None else None, positions=positions.to(DEV) if positions is not None else None)
            assert torch.equal(r, got_q) and torch.equal(a2["k_pages"], a["k_pages"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [([1, 1], [255, 900], 1, 1, 256, 16), ([2, 3, 1], [40, 9, 200], 4, 2, 64, 16), ([17, 30, 1, 0] * 16, [0, 90, 40, 7] * 16, 8, 4, 64, 16),
                                   ([5], [33000], 4, 1, 128, 128)])
def test_a_bound_of_new_tokens_above_the_rows_changes_nothing(shape, dtype):
    """Bit for bit, up to the largest bound that is taken."""
    c = make(*shape, dtype=dtype, seed=61)
    a = on_gpu(c)
    a["max_new"] = c["N"]
    want = paged.paged_attention(**a, return_lse=True)
    k, v = (torch.randn(c["N"], c["Hkv"], c["d"], generator=c["g"]).to(dtype).to(DEV) for _ in range(2))
    pages = {}
    for bound in (c["N"], c["N"] + 1, 1 << 24, (1 << 31) - 1):
        a = on_gpu(c)
        a["max_new"] = bound
        got = paged.paged_attention(**a, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        a.pop("q")
        paged.paged_kv_append(k, v, **a)
        pages[bound] = (a["k_pages"], a["v_pages"])
        assert all(torch.equal(x, y) for x, y in zip(pages[bound], pages[c["N"]]))
    check(c, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_leaves_out_what_has_no_place(dtype):
    c = make([3, 2, 2], [14, 30, 4], 2, 2, 64, 16, dtype, 21)
    c["table"][1, 1] = -1                                  # sequence 1: places 16 .. do not exist
    k, v = (torch.randn(9, 2, 64, generator=c["g"]).to(dtype).to(DEV) for _ in range(2))
    a = on_gpu(c)
    a.pop("q")
    a["lens"][2] = 1                                       # two new tokens in one place: the first is not stored
    before = a["k_pages"].clone()
    rows = torch.tensor([0, 9, 2, 3, 4, 5, -1], dtype=torch.int32, device=DEV)   # tokens 1 and 6 have no source
    tab = modules.rotary_table(16, 64).to(DEV)             # positions 16 .. are not in the table: NaN
    paged.paged_kv_append(k, v, **a, rows=rows, rotary=tab)
    changed = (a["k_pages"].cpu().view(torch.int32 if dtype == torch.float32 else torch.int16)
               != before.cpu().view(torch.int32 if dtype == torch.float32 else torch.int16)).any(-1).any(1).nonzero().tolist()
    t = c["table"]
    # place 14 (page 0) and 16 (page 1) of sequence 0
    assert sorted(map(tuple, changed)) == sorted([(t[0, 0], 14), (t[0, 1], 0)])
    assert torch.isfinite(a["k_pages"][t[0, 0], :, 14]).all() and torch.isnan(a["k_pages"][t[0, 1], :, 0]).all()
    assert torch.isfinite(a["v_pages"][t[0, 1], :, 0]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_prompt_drafts_and_their_verified_path_equal_one_prompt(dtype):
    """As the operators are used together: a prompt enters the cache, a tree of drafts is appended and attends, the accepted path replaces it
    (its positions are the depths), and the next token attends: the same numbers as a chain that never saw the other drafts."""
    g = torch.Generator().manual_seed(31)
    Hq, Hkv, d, page, B = 4, 2, 64, 16, 3
    ctx, total = [21, 40, 3], 8
    tab = modules.rotary_table(64, d).to(DEV)
    pool = [torch.randn(30, Hkv, page, d, generator=g).to(dtype).to(DEV) for _ in range(2)]
    table = torch.arange(30, dtype=torch.int32, device=DEV).view(3, 10)[:, :8].contiguous()
    draw = lambda n: torch.randn(n, Hq + 2 * Hkv, d, generator=g).to(dtype).to(DEV)  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    cu_of = lambda n: i32([0] + list(np.cumsum(n)))  # noqa: E731
    split = lambda f: (f[:, Hq:Hq + Hkv], f[:, Hq + Hkv:], f[:, :Hq])  # noqa: E731
    prompt, drafts, nxt = draw(sum(ctx)), draw(B * total), draw(B)
    k, v, q = split(prompt)
    paged.paged_kv_append(k, v, *pool, table, i32(ctx), cu_of(ctx), max(ctx), rotary=tab)
    # drafts: parent of each of the 8 nodes, the accepted path 0 - 2 - 5 - 7 (depths 0 .. 3), 0 - 2, 0
    parent = [-1, 0, 0, 1, 2, 2, 3, 5]
    depth = [0, 1, 1, 2, 2, 2, 3, 3]
    path = [[0, 2, 5, 7], [0, 2], [0]]
    sees = np.zeros((8, 64), dtype=bool)
    for i, p in enumerate(parent):
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = True
    words = torch.from_numpy(np.packbits(np.tile(sees, (B, 1)), axis=1, bitorder="little").view(np.int64).copy()).to(DEV)
    k, v, q = split(drafts)
    lens = i32([c + total for c in ctx])
    pos = i32([c + dd for c in ctx for dd in depth])
    qr = paged.paged_kv_append(k, v, *pool, table, lens, cu_of([total] * B), total, q=q, rotary=tab, positions=pos)
    out = paged.paged_attention(qr, *pool, table, lens, cu_of([total] * B), total, tree=words)
    n = [len(p) for p in path]
    rows = i32([b * total + j for b, p in enumerate(path) for j in p])
    lens = i32([c + m for c, m in zip(ctx, n)])
    paged.paged_kv_append(k, v, *pool, table, lens, cu_of(n), max(n), rotary=tab, rows=rows)
    k1, v1, q1 = split(nxt)
    lens1 = lens + 1
    q1 = paged.paged_kv_append(k1, v1, *pool, table, lens1, cu_of([1] * B), 1, q=q1, rotary=tab)
    out1 = paged.paged_attention(q1, *pool, table, lens1, cu_of([1] * B), 1)
    # the same sequences, never drafted: the prompt, the path and the next token in one call
    parts, m = [], [c + x + 1 for c, x in zip(ctx, n)]
    at = np.concatenate([[0], np.cumsum(ctx)])
    for b in range(B):
        parts += [prompt[at[b]:at[b + 1]], drafts[[b * total + j for j in path[b]]], nxt[b:b + 1]]
    k, v, q = split(torch.cat(parts))
    fresh = [torch.zeros_like(p) for p in pool]
    q = paged.paged_kv_append(k, v, *fresh, table, i32(m), cu_of(m), max(m), q=q, rotary=tab)
    want = paged.paged_attention(q, *fresh, table, i32(m), cu_of(m), max(m))
    end = np.cumsum(m)
    tol = 4e-6 if dtype == torch.float32 else 3 * 2.0 ** -8  # two outputs of the same numbers, each within a rounding of |out| < 4 and a few 1e-7
    for b in range(B):
        assert float((out1[b] - want[end[b] - 1]).abs().max()) <= tol * 4
        for x, j in enumerate(path[b]):
            assert float((out[b * total + j] - want[end[b] - 1 - n[b] + x]).abs().max()) <= tol * 4


def test_two_runs_are_equal_on_another_stream_and_in_a_graph():
    """A captured append + attention serves other lengths, tables and fills; replays equal eager passes bit for bit."""
    news, ctxs = [5, 1, 12, 30], [200, 900, 3000, 17]
    c = make(news, ctxs, 8, 2, 64, 16, torch.bfloat16, 41)
    a = on_gpu(c)
    a["max_new"] = 64
    f = torch.randn(c["N"], 4, 64, generator=c["g"]).bfloat16().to(DEV)
    q = a.pop("q")

    def step():
        paged.paged_kv_append(f[:, :2], f[:, 2:], **a)
        return paged.paged_attention(q, **a, return_lse=True)

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(first, other))
    graphs = []
    for _ in range(2):  # two graphs that run one after the other on two streams
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = step()
        graphs.append((g, held))
    for lens, cu in (([205, 901, 3012, 47], [0, 5, 6, 18, 48]), ([100, 17, 2000, 1], [0, 20, 20, 47, 48]), ([48, 48, 48, 48], [0, 0, 48, 48, 48])):
        a["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        a["cu"].copy_(torch.tensor(cu, dtype=torch.int32))
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, held in graphs:
            assert all(torch.equal(x[:cu[-1]], y[:cu[-1]]) for x, y in zip(held, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_memory_is_seen_whole_by_every_new_token(dtype):
    """Encoder-decoder attention: lens counts the memory alone; an empty memory gives zeros; rows of 16 * 4 + 1 new tokens."""
    c = make([3, 65, 1, 2], [40, 130, 0, 1], 4, 2, 64, 16, dtype, 71, garbage=math.nan)
    a = on_gpu(c)
    a["lens"] -= torch.tensor(c["news"], dtype=torch.int32, device=DEV)
    # the exact form: the same rows, each the last new token of a sequence as long as the memory
    full = dict(c, news=[], lens=[], cu=None)
    for b, n in enumerate(c["news"]):
        full["news"] += [1] * n
        full["lens"] += [int(c["lens"][b]) - n] * n
    full["table"] = np.concatenate([np.repeat(c["table"][b:b + 1], n, 0) for b, n in enumerate(c["news"])])
    full["cu"] = np.arange(c["N"] + 1, dtype=np.int32)
    full["lens"] = np.array(full["lens"])
    check(full, paged.paged_attention(**a, memory=True, return_lse=True))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_calls_without_new_tokens(dtype):
    c = make([0, 0], [5, 0], 2, 1, 32, 16, dtype, 61)
    a = on_gpu(c)
    for max_new in (0, 3):
        a["max_new"] = max_new
        o, l = paged.paged_attention(**a, return_lse=True)
        assert o.shape == (0, 2, 32) and l.shape == (0, 2)
        b = {k: v for k, v in a.items() if k != "q"}
        before = a["k_pages"].clone()
        e = torch.empty(0, 1, 32, dtype=dtype, device=DEV)
        paged.paged_kv_append(e, e, **b, q=torch.empty(0, 2, 32, dtype=dtype, device=DEV), rotary=modules.rotary_table(4, 32).to(DEV))
        paged.paged_kv_append(e, e, **b, rows=torch.zeros(2, dtype=torch.int32, device=DEV))  # nothing to select from
        assert torch.equal(a["k_pages"], before)


def test_a_cache_beyond_32_bit_offsets():
    """Pages behind 2^32 elements of a pool (8.6 GB a side in bf16; only the pages in use are written)."""
    pages, page, H, d = (1 << 32) // (64 * 2 * 64) + 64, 64, 2, 64
    k, v = (torch.empty(pages, H, page, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    c = make([3, 1], [100, 200], 4, 2, d, page, torch.bfloat16, 51)
    real = pages - 1 - np.arange(c["k"].shape[0])     # the small cache's pages live at the far end
    for x, big in (("k", k), ("v", v)):
        big[torch.from_numpy(real.copy()).to(DEV)] = c[x].to(DEV)
    a = on_gpu(c)
    table = torch.from_numpy(np.where(c["table"] >= 0, real[np.maximum(c["table"], 0)], -1).astype(np.int32)).to(DEV)
    a.update(k_pages=k, v_pages=v, page_table=table)
    check(c, paged.paged_attention(**a, return_lse=True))
    f = torch.randn(4, 4, d, generator=c["g"]).bfloat16().to(DEV)
    a.pop("q")
    paged.paged_kv_append(f[:, :2], f[:, 2:], **a)
    assert torch.equal(k[int(table[1, 3]), :, 200 % 64], f[3, :2])
