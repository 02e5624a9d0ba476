"""Times of the serving operators and token scores that perf/operators.py does not list, and of the greedy search that uses them:

    python3 tools/serving_times.py [copy] [memory] [prompts] [scores] [search]

* copy: what copies of several sizes, writing and reading reach, and a large matrix product: the rates that floors are counted at;
* memory: a drafted pass's rows over the projected encoder output, in the pages PagedDecoderState builds and with the heads outermost;
* prompts: the listed prompts' lengths in bf16 and in fp32;
* scores: the forward scores by themselves, behind their backward pass, and with up to 64 alternatives;
* search: beam 1 against greedy search with drafts (the CTC head's, and beam 1's own hypotheses with tokens replaced).

Operators: captured graphs of 12 calls over three sets of inputs in turn, the median of 15 replays by events; ``us`` is one call."""
import os
import random
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import numpy as np
import torch

from s2t_amd import functional as Fn
from s2t_amd import paged
from s2t_amd import s2t_transformer as M
from s2t_amd.sequence_generator import SequenceGenerator

DEV = "cuda"


def per_call(calls):
    """Median time of one of ``calls`` (run in turn, twelve to a graph) in us."""
    for f in calls:
        f()
    torch.cuda.synchronize()
    n = 12 // len(calls)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(n):
            for f in calls:
                f()
    got = []
    for _ in range(15):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        got.append(a.elapsed_time(b) * 1e3 / (n * len(calls)))
    return sorted(got)[len(got) // 2]


def say(text, us, nbytes=0, flops=0):
    print("%-88s %9.2f us%s%s" % (text, us, "  %6.0f GB/s" % (nbytes / us / 1e3) if nbytes else "", "  %6.0f TFLOP/s" % (flops / us / 1e6) if flops else ""),
          flush=True)


def copy():
    for mib in (16, 64, 128, 256, 1024, 4096):
        sets = [(torch.zeros(mib << 20, dtype=torch.uint8, device=DEV), torch.empty(mib << 20, dtype=torch.uint8, device=DEV)) for _ in range(3)]
        say("copy of %d MiB, three pairs in turn" % mib, per_call([lambda x=x, y=y: y.copy_(x) for x, y in sets]), 2 * (mib << 20))
        say("copy of %d MiB, one pair again and again" % mib, per_call([lambda: sets[0][1].copy_(sets[0][0])]), 2 * (mib << 20))
        if mib >= 1024:
            xs = [x.view(torch.float32) for x, _ in sets]
            ys = [y.view(torch.float32) for _, y in sets]
            say("  y = -x of as much", per_call([lambda x=x, y=y: torch.neg(x, out=y) for x, y in zip(xs, ys)]), 2 * (mib << 20))
            say("  filled, only written", per_call([lambda y=y: y.fill_(1.0) for y in ys]), mib << 20)
            say("  largest of all, only read", per_call([lambda x=x: x.amax() for x in xs]), mib << 20)
            del xs, ys
        del sets
    for dtype, n in ((torch.bfloat16, 8192), (torch.float32, 8192)):
        a, b = (torch.randn(n, n, device=DEV).to(dtype) for _ in range(2))
        out = torch.empty_like(a)
        say("product of %d^3, %s" % (n, dtype), per_call([lambda: torch.mm(a, b, out=out)]), 0, 2 * n ** 3)


def memory():
    H, d, page = 4, 64, 16
    for dtype in (torch.bfloat16, torch.float32):
        for B, frames, rows in ((16, 250, 17), (16, 1000, 17), (16, 250, 1), (64, 250, 17)):
            m = -(-frames // page)
            i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
            table, lens, cu = torch.arange(B * m, dtype=torch.int32, device=DEV).view(B, m), i32([frames] * B), i32([rows * b for b in range(B + 1)])
            qs = [torch.randn(B * rows, H, d, device=DEV).to(dtype) for _ in range(3)]
            kvs = [torch.randn(B * m, page, 2, H, d, device=DEV).to(dtype) for _ in range(3)]
            e = kvs[0].element_size()
            moved, flops = 2 * B * frames * H * d * e + 2 * B * rows * H * d * e, 4 * B * rows * frames * H * d
            for what, views in (("as PagedDecoderState lays it out", [(x[:, :, 0].transpose(1, 2), x[:, :, 1].transpose(1, 2)) for x in kvs]),
                                ("heads outermost", [(x[:, :, 0].transpose(1, 2).contiguous(), x[:, :, 1].transpose(1, 2).contiguous()) for x in kvs])):
                calls = [lambda q=q, k=k, v=v: paged.paged_attention(q, k, v, table, lens, cu, rows, memory=True) for q, (k, v) in zip(qs, views)]
                say("memory, %s: %d sentences x %d frames, %d rows each, %s" % (str(dtype)[6:], B, frames, rows, what), per_call(calls), moved, flops)


def prompts():
    r = np.random.RandomState(7 * 6 + 2001)
    spread = lambda lo, hi: np.rint(lo + (hi - lo) * (r.permutation(6) / 5)).astype(int)  # noqa: E731
    new, ctx = spread(700, 2001), spread(0, 1000)
    H, d, page = 8, 64, 64
    lens = new + ctx
    used = -(-lens // page)
    for dtype in (torch.bfloat16, torch.float32):
        sets = []
        for _ in range(3):
            pages = int(used.sum()) + 3
            order, table, at = np.random.permutation(pages), np.full((6, used.max()), -1, dtype=np.int32), 0
            for b, u in enumerate(used):
                table[b, :u] = order[at:at + u]
                at += u
            k, v = (torch.randn(pages, H, page, d, device=DEV).to(dtype) for _ in range(2))
            sets.append((torch.randn(int(new.sum()), H, d, device=DEV).to(dtype), k, v, torch.from_numpy(table).to(DEV),
                         torch.from_numpy(lens.astype(np.int32)).to(DEV), torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).to(DEV)))
        e = sets[0][0].element_size()
        pairs = int((new * ctx + new * (new + 1) // 2).sum())
        say("prompts, %s: %d tokens of 8 heads of 64 over up to %d keys" % (str(dtype)[6:], new.sum(), lens.max()),
            per_call([lambda s=s: paged.paged_attention(*s, int(new.max())) for s in sets]), (2 * int(lens.sum()) + 2 * int(new.sum())) * H * d * e, 4 * pairs * H * d)


def scores():
    for rows, V, dtype, tops in ((8192, 10000, torch.bfloat16, (0, 4, 10, 32, 48, 64)), (2047, 32001, torch.float32, (0, 8, 32, 48, 64))):
        xs = [(torch.randn(rows, (V + 7) // 8 * 8, device=DEV) * 2).to(dtype)[:, :V] for _ in range(3)]
        y = torch.randint(4, V, (rows,), device=DEV)
        y[torch.randperm(rows, device=DEV)[:rows // 8]] = 1
        live = rows - rows // 8
        for top in tops:
            say("scores and entropy, %d x %d %s, %d alternatives" % (rows, V, str(dtype)[6:], top),
                per_call([lambda x=x: Fn.token_logprobs(x, y, top=top, entropy=True, ignore_index=1) for x in xs]), live * V * xs[0].element_size())
        say("  no entropy, no alternatives", per_call([lambda x=x: Fn.token_logprobs(x, y, ignore_index=1) for x in xs]), live * V * xs[0].element_size())
        say("  entropy, the same logits again and again", per_call([lambda: Fn.token_logprobs(xs[0], y, entropy=True, ignore_index=1)]),
            live * V * xs[0].element_size())
        if dtype is torch.bfloat16:
            up = torch.randn(2, rows, device=DEV)

            def both(x):
                leaf = x.detach().requires_grad_()
                r = Fn.token_logprobs(leaf, y, entropy=True, ignore_index=1)
                return torch.autograd.grad([r.logprob, r.entropy], leaf, [up[0], up[1]])
            say("scores, entropy and gradient, %d x %d bf16" % (rows, V), per_call([lambda x=x: both(x) for x in xs]), (live * 2 + rows) * V * 2)


def search():
    torch.manual_seed(1)
    V, B, T, n = 10000, 16, 1000, 60
    task = M.FakeTask(V)
    model = M.S2TTransformerModel.build_model(M.recipe_args(conformer=True, vocab_size=V), task).prepare(torch.float32, DEV)
    model.eval()
    sample = {"net_input": {"src_tokens": torch.randn(B, T, 80, device=DEV), "src_lengths": torch.full((B,), T, device=DEV)}}

    def timed(text, drafts=None, **kw):
        g = SequenceGenerator([model], task.target_dictionary, beam_size=1, max_len_a=0, max_len_b=n, min_len=n, **kw)
        more = {} if drafts is None else {"drafts": drafts}
        g.generate([model], sample, **more)
        took = []
        for _ in range(5):
            torch.cuda.synchronize()
            a = time.perf_counter()
            r = g.generate([model], sample, **more)
            torch.cuda.synchronize()
            took.append((time.perf_counter() - a) * 1e3)
        print("%-60s %7.1f ms (encoder included)%s" % (text, sorted(took)[2], "  %d passes" % g.draft_passes if kw else ""), flush=True)
        return [h[0]["tokens"].tolist() for h in r]

    said = timed("beam 1, %d sentences x %d frames, %d tokens, fp32" % (B, T, n))
    rng = random.Random(1)
    same = lambda got: sum(a == b for a, b in zip(got, said))  # noqa: E731
    got = timed("drafts of the (untrained) CTC head", draft="ctc")
    print("  %d of %d hypotheses the same" % (same(got), B), flush=True)
    for share in (0.0, 0.05, 0.2, 1.0):
        for most in (16, 32):
            drafts = [[rng.randint(4, V - 1) if rng.random() < share else t for t in s[:-1]] for s in said]
            got = timed("drafts with %d %% of the tokens wrong, %d at a time" % (100 * share, most), drafts, draft="ctc", draft_len=most)
            print("  %d of %d hypotheses the same" % (same(got), B), flush=True)


if __name__ == "__main__":
    print(torch.cuda.get_device_name(), flush=True)
    for part in (copy, memory, prompts, scores, search):
        if len(sys.argv) == 1 or part.__name__ in sys.argv[1:]:
            with torch.no_grad() if part is not scores else torch.enable_grad():
                part()
