"""Workloads of the decoder's serving operators and of the token scores, each in a plain form and through the framework.

Three operators belong together in a decoder that verifies drafted tokens (a CTC transcript, a beam, a tree of alternatives):

* ``append``: the keys and values of new tokens go into a paged cache, rotated by their positions on the way where the model
  has rotary positions (the queries are rotated by the same call); with ``select`` only the accepted drafts are taken over;
* ``attend``: attention of the new tokens over the cache, every token seeing the whole prefix and, of the new ones, itself and its
  ancestors in the draft tree (or all earlier ones: a chain);
* ``score``: log probabilities of given tokens, entropies and the best alternatives of every row of logits, with the gradient.

``own = False`` computes them with elementary torch operations in 32 bits, rounded once at the end."""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}
PAD = 1  # the padding index of the framework's dictionaries: such targets have no score
ROTARY_BASE = 10000.0


def listed():
    return [
        # one step of beam search: 4 sentences x 5 hypotheses, the recipes' decoder (4 heads of 64): latency is all there is
        {"name": "append_beam_step_bf16", "op": "append", "dtype": "bf16", "seqs": 20, "new_min": 1, "new_max": 1, "ctx_min": 20,
         "ctx_max": 200, "q_heads": 4, "kv_heads": 4, "dim": 64, "page": 16, "rotary": False, "select": False},
        # prompts of a batch enter the cache: grouped heads with rotary positions, lengths as ragged as they come
        {"name": "append_prompts_rotary_bf16", "op": "append", "dtype": "bf16", "seqs": 32, "new_min": 40, "new_max": 1023,
         "ctx_min": 0, "ctx_max": 300, "q_heads": 16, "kv_heads": 4, "dim": 128, "page": 64, "rotary": True, "select": False},
        # drafts have been verified: the accepted path of each tree (of up to 16 drafted tokens) is taken over, in the parity type
        {"name": "append_accepted_rotary_fp32", "op": "append", "dtype": "fp32", "seqs": 256, "new_min": 1, "new_max": 9,
         "ctx_min": 10, "ctx_max": 500, "q_heads": 8, "kv_heads": 8, "dim": 64, "page": 32, "rotary": True, "select": True},
        # the attention of that beam step
        {"name": "attend_beam_step_bf16", "op": "attend", "dtype": "bf16", "seqs": 20, "new_min": 1, "new_max": 1, "ctx_min": 20,
         "ctx_max": 200, "q_heads": 4, "kv_heads": 4, "dim": 64, "page": 16, "tree": False, "lse": False},
        # a serving batch, one token for each sequence, long and short caches side by side (8 heads of 64: the d = 512 recipes)
        {"name": "attend_serving_bf16", "op": "attend", "dtype": "bf16", "seqs": 128, "new_min": 1, "new_max": 1, "ctx_min": 100,
         "ctx_max": 4000, "q_heads": 8, "kv_heads": 8, "dim": 64, "page": 64, "tree": False, "lse": False},
        # verification of draft trees, up to 32 nodes for each sequence
        {"name": "attend_tree_bf16", "op": "attend", "dtype": "bf16", "seqs": 64, "new_min": 5, "new_max": 32, "ctx_min": 60,
         "ctx_max": 1500, "q_heads": 8, "kv_heads": 8, "dim": 64, "page": 32, "tree": True, "lse": False},
        # one long recording: few rows over a long cache, grouped heads, the statistics kept for a caller that joins parts
        {"name": "attend_long_grouped_bf16", "op": "attend", "dtype": "bf16", "seqs": 1, "new_min": 5, "new_max": 5,
         "ctx_min": 131000, "ctx_max": 131000, "q_heads": 16, "kv_heads": 4, "dim": 128, "page": 256, "tree": False, "lse": True},
        # draft trees in the parity type
        {"name": "attend_tree_fp32", "op": "attend", "dtype": "fp32", "seqs": 24, "new_min": 1, "new_max": 13, "ctx_min": 1,
         "ctx_max": 300, "q_heads": 4, "kv_heads": 4, "dim": 64, "page": 16, "tree": True, "lse": True},
        # prompts (or whole drafted transcripts) attend in one pass
        {"name": "attend_prompts_bf16", "op": "attend", "dtype": "bf16", "seqs": 6, "new_min": 700, "new_max": 2001, "ctx_min": 0,
         "ctx_max": 1000, "q_heads": 8, "kv_heads": 8, "dim": 64, "page": 64, "tree": False, "lse": False},
        # scores of drafted tokens with the alternatives to branch to (vocabulary of the recipes)
        {"name": "score_drafts_bf16", "op": "score", "dtype": "bf16", "rows": 60, "vocab": 10000, "top": 4, "entropy": False,
         "grad": False, "temperature": 1.0},
        # a training batch: token scores and an entropy term with their gradient
        {"name": "score_train_bf16", "op": "score", "dtype": "bf16", "rows": 8192, "vocab": 10000, "top": 0, "entropy": True,
         "grad": True, "temperature": 1.0},
        # forced decoding of references over a large odd vocabulary, with entropies, alternatives and a temperature
        {"name": "score_references_fp32", "op": "score", "dtype": "fp32", "rows": 2047, "vocab": 32001, "top": 8, "entropy": True,
         "grad": False, "temperature": 0.7},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["append", "attend", "attend", "score"])
        kind = rng.choice(["bf16", "bf16", "fp32"])
        if op == "score":
            grad = rng.random() < 0.4
            case = {"op": op, "dtype": kind, "rows": _spread(rng, 1, 8192), "vocab": _spread(rng, 300, 50000), "top": rng.choice([0, 1, 4, 8, 10]),
                    "entropy": rng.random() < 0.6, "grad": grad, "temperature": rng.choice([1.0, 1.0, 0.7, 1.3])}
        else:
            kv = rng.choice([1, 2, 4, 8])
            case = {"op": op, "dtype": kind, "seqs": _spread(rng, 1, 256), "kv_heads": kv, "q_heads": kv * rng.choice([1, 1, 2, 4]),
                    "dim": rng.choice([32, 64, 64, 128]), "page": rng.choice([16, 32, 64, 256])}
            if op == "append":
                top = _spread(rng, 1, 1024)
                select = rng.random() < 0.3
                top = min(top, 16) if select else top
                case |= {"new_min": max(1, top // 3), "new_max": top, "ctx_min": 0, "ctx_max": _spread(rng, 1, 1000),
                         "rotary": rng.random() < 0.6, "select": select}
            else:
                new = _spread(rng, 1, 2000)
                tree = rng.random() < 0.5 and new > 1
                new = min(new, 64) if tree else new
                ctx = _spread(rng, 1, 60000)
                case |= {"new_min": max(1, new // 3), "new_max": new, "ctx_min": ctx // 20, "ctx_max": ctx, "tree": tree,
                         "lse": rng.random() < 0.3}
        if _cost(case) <= most and _room(case) <= 1.5e9:
            return case


def _lengths(case):
    """New tokens and length of the cache in front of them for each sequence: a property of the case, the same for every seed."""
    r = np.random.RandomState(7 * case["seqs"] + case["new_max"])
    spread = lambda lo, hi: np.rint(lo + (hi - lo) * (r.permutation(case["seqs"]) / max(1, case["seqs"] - 1))).astype(np.int64)  # noqa: E731
    if case["seqs"] == 1:
        return np.array([case["new_max"]]), np.array([case["ctx_max"]])
    return spread(case["new_min"], case["new_max"]), spread(case["ctx_min"], case["ctx_max"])


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "score":
        live = case["rows"] - case["rows"] // 8
        cells = live * case["vocab"]
        return {"bytes": cells * e + (case["rows"] * case["vocab"] * e if case["grad"] else 0) + case["rows"] * (16 + 12 * case["top"]),
                "flops": cells * (10 if case["grad"] else 5)}
    new, ctx = _lengths(case)
    n, d, hq, hk = int(new.sum()), case["dim"], case["q_heads"], case["kv_heads"]
    if case["op"] == "append":
        moved = 4 * n * hk * d * e + n * 8
        if case["rotary"]:
            q = 0 if case["select"] else hq
            return {"bytes": moved + 2 * n * q * d * e + 4 * d * int((new + ctx).max()), "flops": 3 * n * (hk + q) * d}
        return {"bytes": moved, "flops": 0}
    pairs = int((new * ctx + new * (new + 1) // 2).sum())
    return {"bytes": 2 * int((new + ctx).sum()) * hk * d * e + 2 * n * hq * d * e + (4 * n * hq if case["lse"] else 0), "flops": 4 * pairs * hq * d}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 5e14)


def _room(case):
    """Bytes of the largest array that the plain form makes."""
    if case["op"] == "score":
        return 4 * case["rows"] * case["vocab"]
    new, ctx = _lengths(case)
    keys = int((new + ctx).max())
    if case["op"] == "append":
        return 4 * case["seqs"] * keys * case["kv_heads"] * case["dim"]
    return 4 * case["seqs"] * keys * max(case["kv_heads"] * case["dim"], case["q_heads"] * int(new.max()))


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def _tree_words(new, r):
    """Ancestor masks of one random tree for each sequence, a node's parent being any earlier node or the prefix itself:
    [tokens, words] int64, bit j of a token's words is set where it sees new token j."""
    top = int(new.max())
    words = (top + 63) // 64
    parent = np.stack([r.randint(-1, i, len(new)) if i else np.full(len(new), -1) for i in range(top)], 1)
    sees = np.zeros((len(new), top, 64 * words), dtype=bool)
    for i in range(top):
        p = parent[:, i]
        sees[:, i] = np.where((p >= 0)[:, None], sees[np.arange(len(new)), np.maximum(p, 0)], False)
        sees[:, i, i] = True
    packed = np.packbits(sees, axis=-1, bitorder="little").view(np.int64)
    return np.concatenate([packed[b, :n] for b, n in enumerate(new)])


def _rotary(positions, dim):
    """Rows of cosines and sines (their halves side by side), angles in 64 bits."""
    angle = np.arange(positions)[:, None] * ROTARY_BASE ** (-np.arange(0, dim, 2) / dim)[None, :]
    return torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32))


def _cache(case, keys, g, r, kind):
    """A cache in use: its pages scattered over the pool, the table's unused places -1."""
    page = case["page"]
    used = -(-keys // page)
    pages = int(used.sum()) + 3
    table = np.full((case["seqs"], int(used.max())), -1, dtype=np.int32)
    order, at = r.permutation(pages), 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    shape = (pages, case["kv_heads"], page, case["dim"])
    k, v = (torch.randn(shape, generator=g, device="cuda").to(kind) for _ in range(2))
    return k, v, torch.from_numpy(table).cuda()


def prepare(case, seed):
    r = np.random.RandomState(seed % (1 << 32))
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = TYPES[case["dtype"]]
    if case["op"] == "score":
        n, V = case["rows"], case["vocab"]
        # the framework pads its logits' rows to 8 elements; a trained model's rows are peaked, on the target more often than not
        logits = torch.randn(n, (V + 7) // 8 * 8, generator=g, device="cuda") * 2.0
        tokens = torch.randint(4, V, (n,), generator=g, device="cuda")
        logits[torch.arange(n, device="cuda"), tokens] += 6.0 * torch.rand(n, generator=g, device="cuda")
        tokens[torch.from_numpy(r.permutation(n)[:n // 8].copy()).cuda()] = PAD
        up = torch.randn(2 + case["top"], n, generator=g, device="cuda")
        return {"case": case, "logits": logits.to(kind)[:, :V], "tokens": tokens, "up": up}
    new, ctx = _lengths(case)
    hq, hk, d, n = case["q_heads"], case["kv_heads"], case["dim"], int(new.sum())
    s = {"case": case, "most": int(new.max())}
    s["k_pages"], s["v_pages"], s["table"] = _cache(case, new + ctx, g, r, kind)
    s["lens"] = torch.from_numpy((new + ctx).astype(np.int32)).cuda()
    s["cu"] = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
    if case["op"] == "attend":
        s["q"] = torch.randn(n, hq, d, generator=g, device="cuda").to(kind)
        s["tree"] = torch.from_numpy(_tree_words(new, r)).cuda() if case["tree"] else None
        return s
    rows = n
    s["rows"] = None
    if case["select"]:  # of the drafts (16 for each sequence) the accepted ones, in ascending order
        drafts = 16
        rows = drafts * case["seqs"]
        pick = np.concatenate([b * drafts + np.sort(r.permutation(drafts)[:m]) for b, m in enumerate(new)])
        s["rows"] = torch.from_numpy(pick.astype(np.int32)).cuda()
    qkv = torch.randn(rows, hq + 2 * hk, d, generator=g, device="cuda").to(kind)  # one fused projection's rows
    s["q"] = qkv[:, :hq] if case["rotary"] and not case["select"] else None
    s["k"], s["v"] = qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    s["rotary"] = _rotary(int((new + ctx).max()), d).cuda() if case["rotary"] else None
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------
def run(s):
    return {"append": _append, "attend": _attend, "score": _score}[s["case"]["op"]](s)


def _places(s, n):
    """Sequence, number within its new tokens and place in the cache of each new token."""
    cu, lens = s["cu"].long(), s["lens"].long()
    t = torch.arange(n, device=cu.device)
    b = (t[:, None] >= cu[None, 1:]).sum(1)
    i = t - cu[b]
    return b, i, lens[b] - (cu[b + 1] - cu[b]) + i


def _turn(x, cos, sin):
    x = x.float()
    a, b = x.chunk(2, -1)
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _append(s):
    if own:
        from s2t_amd import paged

        q = paged.paged_kv_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu"], s["most"], q=s["q"],
                                  rotary=s["rotary"], rows=s["rows"])
    else:
        k, v, q = s["k"], s["v"], s["q"]
        if s["rows"] is not None:
            k, v = k[s["rows"].long()], v[s["rows"].long()]
        b, _, at = _places(s, k.shape[0])
        page, place = s["table"].long()[b, at // s["case"]["page"]], at % s["case"]["page"]
        if s["rotary"] is not None:
            cos, sin = s["rotary"][at].chunk(2, -1)
            k = _turn(k, cos, sin)
            q = _turn(q, cos, sin).to(s["q"].dtype) if q is not None else None
        s["k_pages"][page, :, place] = k.to(s["k_pages"].dtype)
        s["v_pages"][page, :, place] = v
    out = {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    return out | {"q": q} if q is not None else out


def _attend(s):
    case = s["case"]
    if own:
        from s2t_amd import paged

        out = paged.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu"], s["most"], tree=s["tree"],
                                    return_lse=case["lse"])
        return {"out": out[0], "lse": out[1]} if case["lse"] else {"out": out}
    q, B, hk, d, page = s["q"], case["seqs"], case["kv_heads"], case["dim"], case["page"]
    n, hq = q.shape[:2]
    group, most, keys = hq // hk, s["most"], s["table"].shape[1] * page
    b, i, _ = _places(s, n)
    table = s["table"].long().clamp(min=0)
    k, v = (p[table].float().transpose(2, 3).reshape(B, keys, hk, d).transpose(1, 2) for p in (s["k_pages"], s["v_pages"]))
    padded = torch.zeros(B, most, hk, group, d, device=q.device)
    padded[b, i] = q.float().view(n, hk, group, d)
    padded = padded.permute(0, 2, 3, 1, 4).reshape(B, hk, group * most, d)
    scores = (torch.matmul(padded, k.transpose(2, 3)) * d ** -0.5).view(B, hk, group, most, keys)
    lens, counts = s["lens"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    prefix = (lens - counts)[:, None, None]
    key = torch.arange(keys, device=q.device)[None, None, :]
    if s["tree"] is None:
        sees = key <= prefix + torch.arange(most, device=q.device)[None, :, None]
    else:
        words = torch.zeros(B, most, s["tree"].shape[1], dtype=torch.int64, device=q.device)
        words[b, i] = s["tree"]
        j = (key - prefix).clamp(0, 64 * words.shape[2] - 1).expand(B, most, keys)
        sees = (key < prefix) | ((torch.gather(words, 2, j // 64) >> (j % 64)) & 1).bool()
    sees = (sees & (key < lens[:, None, None]))[:, None, None]
    scores = scores.masked_fill(~sees, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hk, group * most, keys), v).view(B, hk, group, most, d) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4)[b, i].reshape(n, hq, d).to(q.dtype)
    if not case["lse"]:
        return {"out": o}
    return {"out": o, "lse": (top + torch.log(total))[..., 0].permute(0, 3, 1, 2)[b, i].reshape(n, hq)}


def _score(s):
    case, logits, tokens, up = s["case"], s["logits"], s["tokens"], s["up"]
    if own:
        from s2t_amd import functional as Fn

        if case["grad"]:
            logits = logits.detach().requires_grad_()
        r = Fn.token_logprobs(logits, tokens, top=case["top"], entropy=case["entropy"], temperature=case["temperature"],
                              ignore_index=PAD)
        out = {"logprob": r.logprob}
        if case["entropy"]:
            out["entropy"] = r.entropy
        if case["top"]:
            out["top_logprob"], out["top_index"] = r.top_logprob, r.top_index
        if case["grad"]:
            outs, ups = [r.logprob], [up[0]]
            if case["entropy"]:
                outs, ups = outs + [r.entropy], ups + [up[1]]
            if case["top"]:
                outs, ups = outs + [r.top_logprob], ups + [up[2:].t()]
            (out["dlogits"],) = torch.autograd.grad(outs, logits, ups)
        return out
    live = tokens != PAD
    raw = logits.float()
    x = raw * (1.0 / case["temperature"])
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    logp, p = x - top - torch.log(total), e / total
    row = torch.arange(len(tokens), device=x.device)
    zero = torch.zeros((), device=x.device)
    out = {"logprob": torch.where(live, logp[row, tokens], zero)}
    if case["entropy"]:
        h = -(p * logp).sum(-1)
        out["entropy"] = torch.where(live, h, zero)
    if case["top"]:
        left, found, column = raw.clone(), [], torch.arange(raw.shape[1], device=x.device)
        for _ in range(case["top"]):  # the largest, the first of equal ones, one after the other
            best = torch.where(left == left.amax(-1, keepdim=True), column, raw.shape[1]).amin(-1)
            left[row, best] = -math.inf
            found.append(best)
        found = torch.stack(found, 1)
        out["top_logprob"] = torch.where(live[:, None], logp.gather(1, found), zero)
        out["top_index"] = torch.where(live[:, None], found, torch.full_like(found, -1))
    if case["grad"]:
        weight = up[0] + (up[2:].sum(0) if case["top"] else 0.0)
        dx = -p * weight[:, None]
        if case["entropy"]:
            dx -= up[1][:, None] * p * (logp + h[:, None])
        dx[row, tokens] += up[0]
        if case["top"]:
            dx.scatter_add_(1, found, up[2:].t())
        out["dlogits"] = torch.where(live[:, None], dx * (1.0 / case["temperature"]), zero).to(logits.dtype)
    return out


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "score":
        return _exact_score(case, s)
    new, ctx = _lengths(case)
    at = np.concatenate([[0], np.cumsum(new)])
    if case["op"] == "append":
        return _exact_append(case, s, new, ctx, at)
    return _exact_attend(case, s, new, ctx, at)


def _exact_append(case, s, new, ctx, at):
    half, page, table = case["dim"] // 2, case["page"], s["table"].cpu().numpy()
    token = np.arange(at[-1])
    seq = np.repeat(np.arange(case["seqs"]), new)
    pos = ctx[seq] + token - at[seq]
    to = torch.from_numpy(table[seq, pos // page].astype(np.int64) * page + pos % page).cuda()
    phase = torch.ones(len(token), 1, half, dtype=torch.complex128, device="cuda")
    if case["rotary"]:  # the table's values, as complex numbers
        t = s["rotary"].double()[torch.from_numpy(pos).cuda()]
        phase = torch.complex(t[:, :half], t[:, half:])[:, None]

    def turned(x):
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * phase
        return torch.cat([z.real, z.imag], -1)

    pick = slice(None) if s["rows"] is None else s["rows"].long()
    out = {}
    for name, rows in (("k_pages", turned(s["k"][pick])), ("v_pages", s["v"][pick].double())):
        pool = s[name].double().transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
        pool.index_copy_(0, to, rows)
        out[name] = pool.view(-1, page, case["kv_heads"], case["dim"]).transpose(1, 2)
    if s["q"] is not None:
        out["q"] = turned(s["q"])
    return out


def _exact_attend(case, s, new, ctx, at):
    page, group, table = case["page"], case["q_heads"] // case["kv_heads"], s["table"].cpu().numpy()
    words = s["tree"].cpu().numpy() if case["tree"] else None
    outs, lses = [], []
    for b in range(case["seqs"]):
        n, keys = int(new[b]), int(new[b] + ctx[b])
        pages = torch.from_numpy(table[b, :-(-keys // page)].astype(np.int64)).cuda()
        k, v = (p[pages].double().permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, case["dim"])[:, :keys].repeat_interleave(group, 0)
                for p in (s["k_pages"], s["v_pages"]))
        q = s["q"][at[b]:at[b + 1]].double().transpose(0, 1)
        hidden = np.zeros((n, keys), dtype=bool)
        if case["tree"]:
            bits = np.unpackbits(np.ascontiguousarray(words[at[b]:at[b + 1]]).view(np.uint8), axis=1, bitorder="little")
            hidden[:, keys - n:] = bits[:, :n] == 0
        else:
            hidden[:, keys - n:] = ~np.tri(n, dtype=bool)
        z = (q @ k.transpose(1, 2)) / math.sqrt(case["dim"])
        z = z.masked_fill(torch.from_numpy(hidden).cuda(), -math.inf)
        outs.append((torch.softmax(z, -1) @ v).transpose(0, 1))
        lses.append(torch.logsumexp(z, -1).t())
    out = {"out": torch.cat(outs)}
    return out | {"lse": torch.cat(lses)} if case["lse"] else out


def _exact_score(case, s):
    live = s["tokens"] != PAD
    leaf = s["logits"].double().requires_grad_(case["grad"])
    logp = torch.log_softmax(leaf / case["temperature"], -1)
    pick = logp.gather(1, s["tokens"][:, None])[:, 0] * live
    out, total = {"logprob": pick}, (pick * s["up"][0]).sum()
    if case["entropy"]:
        h = torch.special.entr(logp.exp()).sum(-1) * live
        out["entropy"], total = h, total + (h * s["up"][1]).sum()
    if case["top"]:
        index = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        best = logp.gather(1, index) * live[:, None]
        total = total + (best * s["up"][2:].t()).sum()
        out["top_logprob"], out["top_index"] = best, index.masked_fill(~live[:, None], -1)
    if case["grad"]:
        (out["dlogits"],) = torch.autograd.grad(total, leaf)
    return {k: v.detach() for k, v in out.items()}
