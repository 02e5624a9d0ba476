"""What the paged cache and the token scores refuse, checked on the CPU (a call that is right in every other way then asks for the GPU)."""
import ctypes as C

import pytest
import torch

from s2t_amd import _lib as L
from s2t_amd import functional as Fn
from s2t_amd import modules as M
from s2t_amd import paged


def _struct_fields(name):
    import re
    src = open(L.HEADER_PATH).read()
    start = src.index("typedef struct %s {" % name) + len("typedef struct %s {" % name)
    body = re.sub(r"/\*.*?\*/", "", src[start:src.index("} %s;" % name)], flags=re.S)
    names = []
    for decl in body.split(";"):
        parts = decl.replace("*", " ").strip().split(",")
        if parts[0].strip():
            names += [parts[0].split()[-1]] + [p.strip() for p in parts[1:]]
    return names


def test_paged_struct_matches_header_field_order():
    """Names in order, and the packed record as the compiler lays the struct out (8-byte fields on 8 bytes)."""
    assert _struct_fields("s2t_paged_args") == L.PAGED_FIELDS
    codes = L.PAGED_ARGS.format.replace("@", "").replace("10i", "i" * 10).replace(" ", "")
    types = {"P": C.c_void_p, "q": C.c_int64, "i": C.c_int32, "f": C.c_float}
    mirror = type("Mirror", (C.Structure,), {"_fields_": [(n, types[c]) for n, c in zip(L.PAGED_FIELDS, codes)]})
    assert len(codes) == len(L.PAGED_FIELDS) and C.sizeof(mirror) == L.PAGED_ARGS.size
    m = mirror.from_buffer_copy(L.PAGED_ARGS.pack(*range(1, 1 + len(codes))))
    assert [int(getattr(m, n) or 0) for n in L.PAGED_FIELDS] == list(range(1, 1 + len(codes)))
    import re
    src = re.sub(r"/\*.*?\*/", "", open(L.HEADER_PATH).read(), flags=re.S)
    body = src[src.index("typedef struct s2t_paged_args {") + len("typedef struct s2t_paged_args {"):src.index("} s2t_paged_args;")]
    got = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        first, *more = decl.split(",")
        kind = "P" if "*" in first else {"int32_t": "i", "int64_t": "q", "float": "f"}[first.split()[0]]
        got += [kind] * (1 + len(more))
    assert "".join(got) == codes


def _good(dtype=torch.float32, B=3, N=5, H=2, Hq=4, d=32, S=16, P=7):
    return dict(k=torch.zeros(N, H, d, dtype=dtype), v=torch.zeros(N, H, d, dtype=dtype), k_pages=torch.zeros(P, H, S, d, dtype=dtype),
                v_pages=torch.zeros(P, H, S, d, dtype=dtype), page_table=torch.zeros(B, 2, dtype=torch.int32),
                lens=torch.ones(B, dtype=torch.int32), cu=torch.zeros(B + 1, dtype=torch.int32), max_new=2)


def _attend(**change):
    a = _good()
    a.pop("k"), a.pop("v")
    a["q"] = torch.zeros(5, 4, 32)
    a.update(change)
    return paged.paged_attention(a.pop("q"), **a)


def _append(**change):
    a = _good()
    a.update(change)
    return paged.paged_kv_append(**a)


def test_good_calls_ask_for_the_gpu():
    for call in (_attend, _append, lambda: _append(rotary=M.rotary_table(8, 32), q=torch.zeros(5, 4, 32)), lambda: _attend(tree=torch.zeros(5, 1, dtype=torch.int64), return_lse=True),
                 lambda: Fn.token_logprobs(torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64), top=3)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


i32 = torch.int32
BAD_CACHE = [
    dict(k_pages=torch.zeros(7, 2, 16, 32, dtype=torch.float16), v_pages=torch.zeros(7, 2, 16, 32, dtype=torch.float16)),
    dict(v_pages=torch.zeros(7, 2, 16, 32, dtype=torch.bfloat16)),
    dict(v_pages=torch.zeros(8, 2, 16, 32)),
    dict(v_pages=torch.zeros(7, 16, 2, 32).transpose(1, 2)),                     # other strides than k_pages
    dict(k_pages=torch.zeros(7, 2, 12, 32), v_pages=torch.zeros(7, 2, 12, 32)),  # not a power of two
    dict(k_pages=torch.zeros(7, 2, 16, 24), v_pages=torch.zeros(7, 2, 16, 24)),
    dict(k_pages=torch.zeros(7, 2, 16, 272), v_pages=torch.zeros(7, 2, 16, 272)),
    dict(k_pages=torch.zeros(7, 2, 16), v_pages=torch.zeros(7, 2, 16)),
    dict(k_pages=torch.zeros(0, 2, 16, 32), v_pages=torch.zeros(0, 2, 16, 32)),
    dict(page_table=torch.zeros(3, 2, dtype=torch.int64)),
    dict(page_table=torch.zeros(3, 0, dtype=i32)),
    dict(page_table=torch.zeros(2, 3, dtype=i32).t()),
    dict(lens=torch.ones(4, dtype=i32)),
    dict(lens=torch.ones(3, dtype=torch.int64)),
    dict(cu=torch.zeros(3, dtype=i32)),
    dict(cu=torch.zeros(8, dtype=i32)[::2]),
    dict(max_new=-1),
    dict(max_new=1 << 31),
    dict(page_table=torch.zeros(0, 2, dtype=i32), lens=torch.ones(0, dtype=i32), cu=torch.zeros(1, dtype=i32)),
]


@pytest.mark.parametrize("change", BAD_CACHE)
def test_bad_caches_are_refused(change):
    for call in (_append, _attend):
        with pytest.raises(ValueError, match="paged cache"):
            call(**change)


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(5, 3, 32)), dict(k=torch.zeros(5, 2, 64)), dict(k=torch.zeros(5, 2, 32, dtype=torch.bfloat16)), dict(k=torch.zeros(5, 64)),
    dict(v=torch.zeros(4, 2, 32)), dict(v=torch.zeros(5, 2, 64)[..., ::2]), dict(q=torch.zeros(5, 3, 32)), dict(q=torch.zeros(4, 4, 32)),
    dict(q=torch.zeros(5, 4, 32), q_out=torch.zeros(5, 2, 32)), dict(q_out=torch.zeros(5, 4, 32)),
    dict(q=torch.zeros(5, 4, 32), rows=torch.zeros(5, dtype=i32)), dict(rows=torch.zeros(5, dtype=torch.int64)), dict(rows=torch.zeros(10, dtype=i32)[::2]),
    dict(positions=torch.zeros(4, dtype=i32)), dict(rows=torch.zeros(3, dtype=i32), positions=torch.zeros(5, dtype=i32)),
    dict(rotary=torch.zeros(9, 24)), dict(rotary=torch.zeros(9, 48)), dict(rotary=torch.zeros(9, 32, dtype=torch.float64)), dict(rotary=torch.zeros(0, 32)),
    dict(rotary=torch.zeros(9, 64)[:, ::2])])
def test_bad_appends_are_refused(change):
    with pytest.raises(ValueError, match="paged cache"):
        _append(**change)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(5, 3, 32)), dict(q=torch.zeros(5, 0, 32)), dict(q=torch.zeros(5, 4, 16)), dict(q=torch.zeros(5, 4, 32, dtype=torch.bfloat16)),
    dict(q=torch.zeros(5, 4, 64)[..., ::2]), dict(out=torch.zeros(5, 4, 16)), dict(out=torch.zeros(4, 4, 32)), dict(tree=torch.zeros(5, 1, dtype=i32)),
    dict(tree=torch.zeros(4, 1, dtype=torch.int64)), dict(tree=torch.zeros(5, 0, dtype=torch.int64)), dict(tree=torch.zeros(2, 5, dtype=torch.int64).t()),
    dict(tree=torch.zeros(5, 1, dtype=torch.int64), memory=True)])
def test_bad_attention_calls_are_refused(change):
    with pytest.raises(ValueError, match="paged cache"):
        _attend(**change)


def test_expanded_targets_are_refused():
    """One place of memory for many rows cannot be written; it can be read."""
    for call, change in ((_attend, dict(out=torch.zeros(1, 4, 32).expand(5, 4, 32))), (_attend, dict(out=torch.zeros(5, 1, 32).expand(5, 4, 32))),
                         (_append, dict(q=torch.zeros(5, 4, 32), q_out=torch.zeros(1, 4, 32).expand(5, 4, 32))),
                         (_append, dict(k_pages=torch.zeros(1, 2, 16, 32).expand(7, 2, 16, 32), v_pages=torch.zeros(1, 2, 16, 32).expand(7, 2, 16, 32)))):
        with pytest.raises(ValueError, match="expanded"):
            call(**change)
    one = torch.zeros(1, 2, 16, 32).expand(7, 2, 16, 32)
    with pytest.raises(RuntimeError, match="GPU only"):
        _attend(k_pages=one, v_pages=one)
    with pytest.raises(RuntimeError, match="GPU only"):  # (a dimension of one row has any stride)
        _attend(q=torch.zeros(1, 4, 32), out=torch.zeros(4, 32).expand(1, 4, 32))


def test_temperatures_that_fp32_cannot_divide_by_are_refused():
    x, y = torch.zeros(4, 9), torch.zeros(4, dtype=torch.int64)
    for t in (1e-40, 1e-320, 1e40):
        with pytest.raises(ValueError, match="temperature"):
            Fn.token_logprobs(x, y, temperature=t)


def test_bad_scores_are_refused():
    x, y = torch.zeros(4, 9), torch.zeros(4, dtype=torch.int64)
    for args, kw in (((x.half(), y), {}), ((x.double(), y), {}), ((x, y.int()), {}), ((x, y[:3]), {}), ((x, y), {"top": 10}), ((x, y), {"top": -1}),
                     ((torch.zeros(4, 99), y), {"top": 65}), ((x, y), {"temperature": 0.0}), ((x, y), {"temperature": -1.0}),
                     ((x, y), {"temperature": float("nan")}), ((x, y), {"temperature": float("inf")}), ((x,), {}), ((torch.zeros(4, 0), y), {}),
                     ((torch.tensor(1.0), torch.tensor(0)), {})):
        with pytest.raises(ValueError, match="token_logprobs"):
            Fn.token_logprobs(*args, **kw)


def test_forward_mode_tangents_are_refused():
    """They would be dropped without a word: by every tensor that may carry one, under no_grad too (which does not switch them off).  At a
    dual level without tangents all is as ever."""
    from torch.autograd import forward_ad as fa

    def dual(*shape):
        return fa.make_dual(torch.zeros(*shape), torch.ones(*shape))

    y = torch.zeros(4, dtype=torch.int64)
    with fa.dual_level():
        calls = [lambda: Fn.token_logprobs(dual(4, 9), y), lambda: Fn.token_logprobs(dual(4, 9), entropy=True), lambda: _attend(q=dual(5, 4, 32)),
                 lambda: _attend(k_pages=dual(7, 2, 16, 32)), lambda: _attend(v_pages=dual(7, 2, 16, 32)), lambda: _append(k=dual(5, 2, 32)),
                 lambda: _append(v=dual(5, 2, 32)), lambda: _append(q=dual(5, 4, 32)), lambda: _append(v_pages=dual(7, 2, 16, 32)),
                 lambda: _append(rotary=dual(8, 32))]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        for call in (_attend, _append, lambda: Fn.token_logprobs(torch.zeros(4, 9), y)):
            with pytest.raises(RuntimeError, match="GPU only"):
                call()


def test_the_c_entries_refuse_before_they_launch():
    lib = L.lib()
    assert lib.s2t_paged_kv_append(None, None) == -1 and lib.s2t_paged_attention(None, None) == -1
    assert lib.s2t_paged_attention(bytes(L.PAGED_ARGS.size), None) == -1
    buf = torch.zeros(64, dtype=torch.float64)
    p = buf.data_ptr()
    p += -p % 16

    def args(**change):
        a = dict(dtype=0, B=1, N=0, max_new=1, q_heads=2, kv_heads=1, dk=32, num_pages=1, page_size=16, table_pages=1, k_pages=p, v_pages=p,
                        p_sp=512, p_sh=512, p_sr=32, page_table=p, table_stride=1, lens=p, cu=p, k=p, k_st=32, k_sh=32, v=p, v_st=32, v_sh=32, q=p,
                        q_st=64, q_sh=32, q_out=p, qo_st=64, qo_sh=32, out=p, o_st=64, o_sh=32, scale=1.0)
        a.update(change)
        return L.PAGED_ARGS.pack(*(a.get(n) or (0.0 if n == "scale" else 0) for n in L.PAGED_FIELDS))

    for entry in (lib.s2t_paged_kv_append, lib.s2t_paged_attention):
        assert entry(args(), None) == 0  # no rows: nothing is launched
        for status, change in ((-2, dict(dtype=2)), (-1, dict(B=0)), (-1, dict(B=65536)), (-1, dict(page_size=24)), (-1, dict(q_heads=3, kv_heads=2)),
                               (-4, dict(dk=24)), (-4, dict(dk=272)), (-1, dict(num_pages=0)), (-1, dict(lens=None)), (-3, dict(k_pages=p + 4)),
                               (-3, dict(p_sr=33)), (-3, dict(q_st=66)), (-4, dict(table_pages=1 << 27))):
            assert entry(args(**change), None) == status, change
    from s2t_amd import kernels as K
    ws = lambda **change: lib.s2t_paged_attention_ws_bytes(args(N=5, max_new=5, **change))  # noqa: E731
    assert ws(table_pages=K.PAGED_ONE_RANGE // 16) == ws(page_size=1, table_pages=K.PAGED_ONE_RANGE) == 0 < ws(table_pages=1 << 16)
    assert lib.s2t_paged_attention(args(N=5, max_new=5, table_pages=1 << 16), None) == -1   # no workspace
    assert lib.s2t_paged_kv_append(args(rows=p), None) == -1            # with q
    assert lib.s2t_paged_kv_append(args(rotary=p, rot_dim=48, rotary_positions=1), None) == -1
    assert lib.s2t_paged_attention(args(tree=p, tree_words=0), None) == -1
    assert lib.s2t_paged_attention(args(tree=p, tree_words=1, memory=1), None) == -1
    f, b = lib.s2t_token_logprobs_fwd, lib.s2t_token_logprobs_bwd
    assert f(0, p, 8, 0, 8, p, -1, 1.0, 0, p, p, p, None, None, None) == 0
    assert f(0, p, 7, 0, 8, p, -1, 1.0, 0, p, p, p, None, None, None) == -1       # rows overlap
    assert f(2, p, 8, 0, 8, p, -1, 1.0, 0, p, p, p, None, None, None) == -2
    assert f(0, p, 99, 0, 99, p, -1, 1.0, 65, p, p, p, p, p, None) == -4
    assert f(0, p, 8, 1, 8, p, -1, 1.0, 2, p, p, p, None, p, None) == -1
    assert f(0, p, 8, 1, 8, None, -1, 1.0, 0, p, p, p, None, None, None) == -1    # a score without a token
    assert b(0, p, 8, 0, 8, p, -1, 1.0, 0, p, None, p, None, None, None, p, 8, None) == 0
    assert b(0, p, 8, 1, 8, p, -1, 1.0, 0, p, None, p, p, None, None, p, 8, None) == -1   # g_entropy without the entropy
    assert b(0, p, 8, 1, 8, p, -1, 1.0, 2, p, None, None, None, p, None, p, 8, None) == -1  # g_top without the columns


def test_a_bound_of_new_tokens_above_the_rows_counts_as_the_rows():
    """It neither overflows nor changes how a call is cut (the workspace shows that); more tokens than a launch takes are refused."""
    lib = L.lib()
    buf = torch.zeros(64, dtype=torch.float64)
    p = buf.data_ptr()
    p += -p % 16

    def args(N, max_new, **change):
        a = dict(dtype=0, B=1, N=N, max_new=max_new, q_heads=2, kv_heads=1, dk=32, num_pages=1, page_size=16, table_pages=1 << 16, k_pages=p, v_pages=p,
                 p_sp=512, p_sh=512, p_sr=32, page_table=p, table_stride=1, lens=p, cu=p, k=p, k_st=32, k_sh=32, v=p, v_st=32, v_sh=32, q=p,
                 q_st=64, q_sh=32, q_out=p, qo_st=64, qo_sh=32, out=p, o_st=64, o_sh=32, scale=1.0)
        a.update(change)
        return L.PAGED_ARGS.pack(*(a.get(n) or (0.0 if n == "scale" else 0) for n in L.PAGED_FIELDS))

    for N in (1, 5, 40, 700):
        for change in ({}, dict(q_heads=8), dict(dk=128, q_st=256, q_sh=128, p_sr=128), dict(B=9)):
            tight = lib.s2t_paged_attention_ws_bytes(args(N, N, **change))
            assert tight > 0 or N * change.get("B", 1) > 4096   # (enough rows: no ranges)
            for loose in (N + 1, 64 * N, 1 << 20, (1 << 31) - 1):
                assert lib.s2t_paged_attention_ws_bytes(args(N, loose, **change)) == tight
                assert tight == 0 or lib.s2t_paged_attention(args(N, loose, **change), None) == -1   # no workspace
    for entry in (lib.s2t_paged_kv_append, lib.s2t_paged_attention):
        assert entry(args(0, (1 << 31) - 1), None) == 0
        assert entry(args((1 << 31) - 1, (1 << 31) - 1), None) == -4


def test_pages_are_dealt_out_and_come_back():
    c = paged.PagedKVCache(2, 3, 5, 4, 1, 16, torch.float32, "cpu", page_size=8)
    c.reserve(0, 9)
    c.reserve(1, 8)
    c.reserve(0, 16)  # has them
    assert c.host_table.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1], [-1] * 4] and c.table.max() == -1
    c.sync()
    assert torch.equal(c.table, c.host_table) and not c.dirty
    with pytest.raises(RuntimeError, match="3 more pages"):
        c.reserve(2, 24)
    c.release(0)
    c.reserve(2, 24)
    assert sorted(c.held[2]) == [0, 1, 3] and c.host_table[0].max() == -1
    with pytest.raises(RuntimeError, match="its table's row takes"):
        c.reserve(2, 40)


def test_rotary_table():
    t = M.rotary_table(5, 32)
    assert t.shape == (5, 32) and torch.equal(t[0], torch.cat([torch.ones(16), torch.zeros(16)]))
    far = M.rotary_table(100001, 32)[100000].double()
    w = 10000.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64) / 32)
    assert float((far - torch.cat([torch.cos(1e5 * w), torch.sin(1e5 * w)])).abs().max()) < 2.0 ** -24


def test_drafted_sentences_say_what_the_decoder_says():
    """The bookkeeping of greedy search with drafts against a decoder that is a table: whatever the draft, the output is the decoder's, the
    kept nodes spell it, and a tree's words hold each node's ancestors."""
    import random

    from s2t_amd.sequence_generator import _DraftedSentence, _words

    assert _words(1, 1) == [1] and _words(1 << 63, 1) == [-(1 << 63)] and _words((1 << 64) | 5, 2) == [5, 1] and _words((1 << 128) - 1, 2) == [-1, -1]
    rng = random.Random(3)
    for case in range(300):
        said = [rng.randint(4, 9) for _ in range(rng.randint(0, 30))] + [2]
        draft = list(said[:-1])
        for _ in range(rng.randint(0, 6)):
            i = rng.randint(0, len(draft))
            kind = rng.random()
            if kind < 0.4 and i < len(draft):
                draft[i] = rng.randint(4, 9)
            elif kind < 0.7 and i < len(draft):
                del draft[i]
            else:
                draft.insert(i, rng.randint(4, 9))
        max_len = len(said) - 1 + rng.randint(0, 3)
        s = _DraftedSentence(draft, 2)
        cache, passes = [], 0
        while not s.done:
            passes += 1
            s.plan(rng.randint(1, 8), max_len)
            assert max(n.depth for n in s.nodes) + s.kept <= max_len
            before = [2] + said[:s.kept]
            choices = []
            for i, n in enumerate(s.nodes):
                up = [j for j in range(len(s.nodes)) if n.sees >> j & 1]
                assert up[-1] == i and [s.nodes[j].depth for j in up] == list(range(n.depth + 1))
                spelt = cache + [s.nodes[j].token for j in up]
                agrees = spelt == ([2] + said)[:len(spelt)]
                choices.append((said[len(spelt) - 1], -0.5) if agrees else (rng.randint(4, 9), -9.0))
            assert s.branches or all(n.sees == (2 << i) - 1 for i, n in enumerate(s.nodes))
            path = s.walk(choices)
            cache += [s.nodes[i].token for i in path]
            assert cache == before + said[len(before) - 1:][:len(cache) - len(before)] and len(cache) == s.kept
        assert s.out == said and len(s.scores) == len(said) and passes <= len(said)
    s = _DraftedSentence(list(range(4, 24)), 2)   # a right draft of 20 tokens, 8 at a time: 9 said in the first pass, 9, then the rest
    said, passes = list(range(4, 24)) + [2], 0
    while not s.done:
        s.plan(8, 40)
        s.walk([(said[s.kept + n.depth], 0.0) for n in s.nodes])
        passes += 1
    assert s.out == said and passes == 3
