"""Paged key/value cache of an incremental decoder and attention of several new tokens of a sequence over it.

The reference's decoder keeps one dense key/value buffer per layer, takes one token per pass and copies the buffers when hypotheses change
places (modules/multihead_attention.py:302-339,574-592).  Here the memory of a layer is a pool of pages that a table deals out to
sequences, and a pass may bring any number of new tokens to each of them: a prompt, the next token, or DRAFTED tokens — a chain
(a CTC transcript) or a tree of alternatives — of which the accepted ones are taken over afterwards.

All functions work on the tensors a serving program keeps:

* ``k_pages`` / ``v_pages`` ``[pages, kv_heads, page_size, head_dim]`` float32 or bfloat16, last dimension contiguous, equal strides (a
  permuted view of ``[pages, page_size, kv_heads, head_dim]`` will do); page_size a power of two, head_dim a multiple of 16 up to 256;
* ``page_table`` ``[seqs, n]`` int32: page of the places ``i * page_size ..`` of each sequence; unused entries may hold anything;
* ``lens`` ``[seqs]`` int32: length of each sequence INCLUDING its new tokens;
* ``cu`` ``[seqs + 1]`` int32: the new tokens' rows of sequence b are ``cu[b] .. cu[b + 1] - 1``, the last one at place ``lens[b] - 1``;
* ``max_new``: no sequence brings more new tokens than this (a launch bound: later ones of a sequence are left out; a loose one costs empty
  workgroups, above the number of rows it counts as that).

What table, lens, cu, tree, positions and rows say is read on the device, so a captured graph serves batches of any fill; rows behind the
last sequence are left as they were, and an entry that leads out of its bounds is never followed (include/s2t_hip.h).
"""
import torch

from . import _lib as L
from . import kernels as K

_TYPES = {torch.float32: L.S2T_F32, torch.bfloat16: L.S2T_BF16}
_I32 = torch.int32


_NONE3 = (0, 0, 0)
_NO_KV, _NO_APPEND, _NO_ATTENTION = (0,) * 6, (0,) * 9, (0, 0, 0, 0, 0, 0, 0, 0.0, 0, 0, 0)  # fields of s2t_paged_args that a call leaves out


def _refuse(what):
    raise ValueError("paged cache: " + what)


def _check_cache(k_pages, v_pages, page_table, lens, cu, max_new):
    """Raises for what is wrong with a cache."""
    if k_pages.dim() != 4 or k_pages.dtype not in _TYPES or v_pages.dtype != k_pages.dtype or v_pages.shape != k_pages.shape:
        _refuse("k_pages and v_pages must be [pages, kv_heads, page_size, head_dim] of one type (float32 or bfloat16), got %s %s and %s %s" % (
            tuple(k_pages.shape), k_pages.dtype, tuple(v_pages.shape), v_pages.dtype))
    if k_pages.stride() != v_pages.stride() or k_pages.stride(3) != 1:
        _refuse("k_pages and v_pages need equal strides and a contiguous last dimension")
    P, H, S, d = k_pages.shape
    if P < 1 or H < 1 or S < 1 or S & (S - 1) or d % 16 or not 16 <= d <= 256:
        _refuse("page_size must be a power of two and head_dim a multiple of 16 up to 256, got %s" % (tuple(k_pages.shape),))
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[1] < 1 or (page_table.stride(1) != 1 and page_table.shape[1] > 1):
        _refuse("page_table must be int32 [seqs, pages of a sequence] with contiguous rows")
    B = page_table.shape[0]
    if lens.dtype != torch.int32 or tuple(lens.shape) != (B,) or not lens.is_contiguous():
        _refuse("lens must be int32 [%d], contiguous" % B)
    if cu.dtype != torch.int32 or tuple(cu.shape) != (B + 1,) or not cu.is_contiguous():
        _refuse("cu must be int32 [%d], contiguous" % (B + 1))
    if not 1 <= B <= 65535 or not 0 <= max_new < 1 << 31:
        _refuse("1 to 65535 sequences and 0 <= max_new < 2^31 expected, got %d and %s" % (B, max_new))


def _cache_fields(k_pages, v_pages, page_table, lens, cu, max_new, N, q_heads):
    """-> the fields of s2t_paged_args up to cu.  One look at everything; what fails it is named by _check_cache."""
    kind, shape, stride = k_pages.dtype, k_pages.shape, k_pages.stride()
    of_table = page_table.shape
    if len(shape) == 4 and len(of_table) == 2:
        P, H, S, d = shape
        B, n = of_table
        row, step = page_table.stride()
        if (kind in _TYPES and v_pages.dtype is kind and v_pages.shape == shape and v_pages.stride() == stride and stride[3] == 1
                and P > 0 and H > 0 and S > 0 and not S & (S - 1) and not d & 15 and 16 <= d <= 256 and n > 0 and 0 < B < 65536
                and page_table.dtype is lens.dtype is cu.dtype is _I32 and (step == 1 or n == 1)
                and lens.shape == (B,) and cu.shape == (B + 1,) and lens.is_contiguous() and cu.is_contiguous() and 0 <= max_new < 1 << 31
                and N < 1 << 31):
            if q_heads < 1 or q_heads % H:
                _refuse("%d query heads over %d key/value heads" % (q_heads, H))
            return (_TYPES[kind], B, N, max_new, q_heads, H, d, P, S, n, k_pages.data_ptr(), v_pages.data_ptr(), stride[0], stride[1],
                    stride[2], page_table.data_ptr(), row, lens.data_ptr(), cu.data_ptr())
    _check_cache(k_pages, v_pages, page_table, lens, cu, max_new)
    _refuse("%d rows" % N)


def _rows(name, t, heads, kind, d, n=None):
    """-> address and strides of [n, heads, d]."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or t.dtype is not kind or shape[2] != d or stride[2] != 1 or (heads is not None and shape[1] != heads) \
            or (n is not None and shape[0] != n):
        _refuse("%s must be [%s, %s, %d] %s with a contiguous last dimension, got %s %s" % (
            name, "rows" if n is None else n, "heads" if heads is None else heads, d, kind, tuple(shape), t.dtype))
    return t.data_ptr(), stride[0], stride[1]


def _no_overlap(name, t):
    if any(n > 1 and step == 0 for n, step in zip(t.shape, t.stride())):
        _refuse("%s to be written may not be expanded, got strides %s" % (name, t.stride()))


def _target(name, t, heads, kind, d, n):
    """``_rows`` of a tensor that is written."""
    of = _rows(name, t, heads, kind, d, n)
    if not (of[1] and of[2]):
        _no_overlap(name, t)
    return of


def _like(q):
    """-> a new tensor of q's shape, its address and strides."""
    t = torch.empty_like(q)
    stride = t.stride()
    return t, (t.data_ptr(), stride[0], stride[1])


def _index(name, t, n):
    if t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous():
        _refuse("%s must be int32 [%d], contiguous" % (name, n))
    return t.data_ptr()


def _device(k_pages, v_pages, page_table, lens, cu, x, others):
    """-> index of the one device that all of them live on; ``x``: the rows that come first."""
    L.refuse_tangents("paged cache", k_pages, v_pages, x, *others)
    dev = k_pages.get_device()
    same = dev == v_pages.get_device() == page_table.get_device() == lens.get_device() == cu.get_device() == x.get_device() and dev >= 0
    grad = x.requires_grad or k_pages.requires_grad or v_pages.requires_grad
    for t in others:
        same = same and t.get_device() == dev
        grad = grad or t.requires_grad
    if not same:
        tensors = (k_pages, v_pages, page_table, lens, cu, x, *others)
        L.require_cuda(*tensors)
        _refuse("tensors on several devices: %s" % ", ".join(str(t.device) for t in tensors))
    if grad and torch.is_grad_enabled():
        raise RuntimeError("the paged cache is inference only: wrap the decoder in torch.no_grad()")
    return dev


def paged_kv_append(k, v, k_pages, v_pages, page_table, lens, cu, max_new, q=None, rotary=None, positions=None, rows=None, q_out=None):
    """Stores the new tokens' keys and values ``[N, kv_heads, head_dim]`` (views of a fused projection's rows are read in place; they may
    not lie in the pages themselves, nor q_out where k or v do).

    ``rotary`` (float32 ``[positions, rot_dim]``: cosines, then sines; ``modules.rotary_table``) turns the first rot_dim elements of every
    key by the token's place, or by ``positions[t]`` (int32: in a tree of drafts the depth, not the place), element i together with
    element i + rot_dim / 2; a position outside the table is stored as NaN.  ``q`` ``[N, q_heads, head_dim]`` is turned by the same call
    into ``q_out`` (default: a new tensor; ``q`` itself: in place) and returned.
    ``rows`` (int32 [N], instead of q): new token t takes row ``rows[t]`` of k and v — the accepted drafts of a verified tree, whose
    projections the caller has kept; a row outside k is not stored."""
    src = k.shape[0] if k.dim() else 0
    N = src if rows is None else rows.shape[0] if rows.dim() else -1
    cache = _cache_fields(k_pages, v_pages, page_table, lens, cu, max_new, N, k_pages.shape[1] if q is None else q.shape[1] if q.dim() > 1 else 0)
    kind, H, d = k_pages.dtype, cache[5], cache[6]
    if not (cache[12] and cache[13] and cache[14]):
        _no_overlap("k_pages and v_pages", k_pages)
    kf = _rows("k", k, H, kind, d)
    vf = _rows("v", v, H, kind, d, src)
    others = [v]
    qf = of = turn = _NONE3
    at = pick = 0
    if q is not None:
        if rows is not None:
            _refuse("q cannot be turned together with a selection of rows")
        qf = _rows("q", q, None, kind, d, N)
        q_out, of = _like(q) if q_out is None else (q_out, _target("q_out", q_out, cache[4], kind, d, N))
        others += (q, q_out)
    elif q_out is not None:
        _refuse("q_out without q")
    if rotary is not None:
        if rotary.dtype is not torch.float32 or rotary.dim() != 2 or not rotary.is_contiguous() or rotary.shape[0] < 1 \
                or rotary.shape[1] % 16 or not 16 <= rotary.shape[1] <= d:
            _refuse("rotary must be float32 [positions, rot_dim], contiguous, rot_dim a multiple of 16 up to head_dim, got %s %s" % (
                tuple(rotary.shape), rotary.dtype))
        turn = (rotary.data_ptr(), *rotary.shape)
        others.append(rotary)
    if positions is not None:
        at = _index("positions", positions, N)
        others.append(positions)
    if rows is not None:
        pick = _index("rows", rows, N)
        others.append(rows)
    K.paged_kv_append(_device(k_pages, v_pages, page_table, lens, cu, k, others),
                      L.PAGED_ARGS.pack(*cache, *kf, *vf, *qf, *of, *turn, at, pick, src, *_NO_ATTENTION))
    return q_out


def paged_attention(q, k_pages, v_pages, page_table, lens, cu, max_new, tree=None, scale=None, out=None, return_lse=False, memory=False):
    """``softmax(scale * q k^T) v`` of the new tokens ``q [N, q_heads, head_dim]`` over their sequences' pages (the new tokens' own keys and
    values have been appended): query head h reads key/value head ``h // (q_heads // kv_heads)``.

    Every new token sees the whole prefix.  Of the new tokens of its sequence it sees those up to itself, or with ``tree`` (int64
    ``[N, words]``) new token j where bit ``j % 64`` of word ``j // 64`` of its row is set — its ancestors and itself, any other set will do.
    With ``memory`` the pages hold something the new tokens only read (the projected encoder output of an encoder-decoder attention): lens
    counts its places alone, and every new token sees all of them.
    A row that sees nothing comes out 0 with lse -inf; what a row does not see never touches it, infinities and NaN included.
    Inference only.  -> out [N, q_heads, head_dim] (``out`` if given), with ``return_lse`` also the fp32 logsumexp [N, q_heads]."""
    shape = q.shape
    N, Hq = shape[:2] if len(shape) == 3 else (0, 0)
    cache = _cache_fields(k_pages, v_pages, page_table, lens, cu, max_new, N, Hq)
    kind, d = k_pages.dtype, cache[6]
    qf = _rows("q", q, Hq, kind, d)
    bits, others = _NONE3, ()
    if tree is not None:
        if memory:
            _refuse("a tree over a memory that holds no new tokens")
        if tree.dtype is not torch.int64 or tree.dim() != 2 or tree.shape[0] != N or tree.shape[1] < 1 or (tree.stride(1) != 1 and tree.shape[1] > 1):
            _refuse("tree must be int64 [%d, words] with contiguous rows, got %s %s" % (N, tuple(tree.shape), tree.dtype))
        bits = (tree.data_ptr(), tree.stride(0), tree.shape[1])
        others = (tree,)
    if out is None:
        out, of = _like(q)
    else:
        of = _target("out", out, Hq, kind, d, N)
        others += (out,)
    dev = _device(k_pages, v_pages, page_table, lens, cu, q, others)
    lse, to_lse = None, 0
    if return_lse:
        lse = torch.empty(N, Hq, dtype=torch.float32, device=q.device)
        to_lse = lse.data_ptr()
    scale = d ** -0.5 if scale is None else float(scale)
    pack = L.PAGED_ARGS.pack
    args = pack(*cache, *_NO_KV, *qf, *_NO_APPEND, *of, to_lse, *bits, scale, 1 if memory else 0, 0, 0)
    if cache[8] * cache[9] > K.PAGED_ONE_RANGE:
        n = K.paged_attention_ws_bytes(args)
        if n > 0:  # from the allocator: a captured graph keeps its own, another stream gets another
            ws = torch.empty(n, dtype=torch.uint8, device=q.device)
            args = pack(*cache, *_NO_KV, *qf, *_NO_APPEND, *of, to_lse, *bits, scale, 1 if memory else 0, ws.data_ptr(), n)
    K.paged_attention(dev, args)
    return (out, lse) if return_lse else out


class PagedKVCache:
    """Pages of ``layers`` decoder layers and the table that deals them out: a sequence takes pages as it grows (``reserve``) and gives them
    back when it is done (``release``).  ``k[l]`` / ``v[l]`` are layer l's pages, ``table`` the tensor the functions above take; its rows
    change on the host and reach the device with the next ``sync``."""

    def __init__(self, layers, seqs, pages, pages_per_seq, kv_heads, head_dim, dtype, device, page_size=16):
        self.page_size, self.pages_per_seq = page_size, pages_per_seq
        self.k, self.v = (torch.empty(layers, pages, kv_heads, page_size, head_dim, dtype=dtype, device=device) for _ in range(2))
        self.host_table = torch.full((seqs, pages_per_seq), -1, dtype=torch.int32)
        self.table = self.host_table.to(device, copy=True)
        self.free = list(range(pages - 1, -1, -1))
        self.held = [[] for _ in range(seqs)]
        self.dirty = False

    def reserve(self, seq, places):
        """Pages for the first ``places`` places of a sequence."""
        need = -(-places // self.page_size) - len(self.held[seq])
        if need <= 0:
            return
        if need > len(self.free) or len(self.held[seq]) + need > self.pages_per_seq:
            raise RuntimeError("paged cache: sequence %d needs %d more pages, %d are free and %d its table's row takes" % (
                seq, need, len(self.free), self.pages_per_seq - len(self.held[seq])))
        for _ in range(need):
            self.host_table[seq, len(self.held[seq])] = self.free[-1]
            self.held[seq].append(self.free.pop())
        self.dirty = True

    def release(self, seq):
        """All pages of a sequence are free again."""
        self.free += reversed(self.held[seq])
        self.held[seq] = []
        self.host_table[seq] = -1
        self.dirty = True

    def sync(self):
        if self.dirty:
            self.table.copy_(self.host_table)
            self.dirty = False
