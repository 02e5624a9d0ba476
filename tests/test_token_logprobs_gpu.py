"""functional.token_logprobs (csrc/token_logprobs.hip): log probabilities of given tokens, entropies, best alternatives and their gradient
against the definitions in float64 on the CPU.

Bounds.  Let e = 2^-24 (half a step of fp32), z = logits / T.  Rounding z costs e |z|; the differences z - m and z - lse each cost half
a step of a number below 2 max|z|; the hardware exponential and logarithm stay within 2 steps, the exponential also turns the rounding
of its scaled argument (below 2 max|z|) into a relative error of as much; a sum of V positive terms accumulated in at most V / 64 + 32 serial steps
costs e for each.  So every log probability is within EP = e (8 max|z| + V / 64 + 64) of the exact one, and a probability within EP of
itself.  The entropy sum p |log p| then moves by EP (2 H + 2), a gradient by what its factors move, and results held in bf16 by half a
step, 2^-8 of the value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from s2t_amd import functional as Fn  # noqa: E402

DEV = "cuda"
E = 2.0 ** -24


def _logits(rows, V, dtype, seed, pad=True, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    ld = (V + 7) // 8 * 8 if pad else V
    x = (torch.randn(rows, ld, generator=g) * scale).to(dtype)
    return x.to(DEV)[:, :V], g


def _exact(x, tokens, top, T, ignore=None, ups=None):
    """x: float tensor on the CPU -> (logprob, entropy, top_lp, top_idx, gradient of the weighted sum, max|z|) in float64"""
    leaf = x.double().requires_grad_()
    lp = torch.log_softmax(leaf / T, -1)
    p = lp.exp()
    live = torch.ones(x.shape[0], dtype=torch.bool) if ignore is None else tokens != ignore
    at = tokens.clamp(0, x.shape[1] - 1)
    pick = torch.where(live, lp.gather(1, at[:, None])[:, 0], 0.0)
    h = torch.where(live, -torch.where(p > 0, p * lp, 0.0).sum(-1), 0.0)
    idx = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :top]
    best = torch.where(live[:, None], lp.gather(1, idx), 0.0)
    grad = None
    if ups is not None:
        total = sum((o * u.double()).sum() for o, u in zip((pick, h, best), ups) if u is not None)
        (grad,) = torch.autograd.grad(total, leaf)
    return pick.detach(), h.detach(), best.detach(), idx.masked_fill(~live[:, None], -1), grad, p.detach(), lp.detach()


def _ep(x, T):
    z = x.double() / T
    return E * (8 * float(z[z.isfinite()].abs().max()) + x.shape[1] / 64 + 64)


SIZES = [(1, 1, 1), (1, 2, 2), (3, 7, 7), (5, 64, 3), (4, 257, 64), (17, 1000, 8), (60, 10000, 4), (3, 32001, 10), (2, 70001, 64), (700, 300, 1), (9, 2561, 12), (5, 5121, 30), (130, 4000, 5)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,top", SIZES)
@pytest.mark.parametrize("T", [1.0, 0.7])
def test_scores_and_gradient_against_float64(rows, V, top, dtype, T):
    x, g = _logits(rows, V, dtype, rows * 31 + V)
    tokens = torch.randint(0, V, (rows,), generator=g)
    if rows > 2:
        tokens[1] = -7  # ignored
    ups = [torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn(rows, top, generator=g)]
    leaf = x.detach().requires_grad_()
    r = Fn.token_logprobs(leaf, tokens.to(DEV), top=top, entropy=True, temperature=T, ignore_index=-7)
    (dx,) = torch.autograd.grad([r.logprob, r.entropy, r.top_logprob], leaf, [u.to(DEV) for u in ups])
    xc = x.float().cpu()
    lp, h, best, idx, grad, p, alllp = _exact(xc, tokens, top, T, -7, ups)
    ep = _ep(xc, T)
    assert torch.equal(r.top_index.cpu(), idx)
    assert float((r.logprob.cpu().double() - lp).abs().max()) <= ep
    assert float((r.top_logprob.cpu().double() - best).abs().max()) <= ep
    assert bool(((r.entropy.cpu().double() - h).abs() <= ep * (2 * h + 2)).all())
    half = E if dtype == torch.float32 else 2.0 ** -8
    W = ups[0].abs().double() + ups[2].abs().double().sum(1)
    gh = ups[1].abs().double()[:, None]
    inner = W[:, None] + gh * (alllp.abs() + h[:, None])
    sparse = torch.zeros_like(p).scatter_add_(1, tokens.clamp(0)[:, None], ups[0].abs().double()[:, None])
    sparse.scatter_add_(1, idx.clamp(0), ups[2].abs().double())
    # p moves by ep of itself, log p + H by ep (2 H + 3); the products, the sum of the upstream gradients and the last add by a few e
    bound = half * grad.abs() + (1 / T) * (p * inner * (ep + (top + 8) * E) + p * gh * ep * (2 * h[:, None] + 3) + 4 * E * sparse)
    bound = bound + 1.2e-38  # the smallest normal fp32 number: smaller results may be flushed
    assert bool(((dx.cpu().double() - grad).abs() <= bound).all())
    if rows > 2:
        assert not dx[1].any() and float(r.logprob[1]) == 0.0 and float(r.entropy[1]) == 0.0 and int(r.top_index[1, 0]) == -1


def test_gradient_against_differences():
    x, g = _logits(3, 41, torch.float32, 5, scale=1.0)
    tokens = torch.tensor([4, 40, 0])
    up = [torch.randn(3, generator=g), torch.randn(3, generator=g), torch.randn(3, 5, generator=g)]
    leaf = x.detach().requires_grad_()
    r = Fn.token_logprobs(leaf, tokens.to(DEV), top=5, entropy=True, temperature=1.3)
    (dx,) = torch.autograd.grad([r.logprob, r.entropy, r.top_logprob], leaf, [u.to(DEV) for u in up])

    def value(y):
        lp, h, best, _, _, _, _ = _exact(y, tokens, 5, 1.3)
        return float((lp * up[0]).sum() + (h * up[1]).sum() + (best * up[2]).sum())

    step = 1e-5
    base = x.double().cpu()
    for r_, c in ((0, 4), (0, 11), (1, 40), (1, 3), (2, 0), (2, 17)):
        hi, lo = base.clone(), base.clone()
        hi[r_, c] += step
        lo[r_, c] -= step
        # central differences in 64 bits: truncation step^2 times a third derivative of order 10, rounding 1e-15 / step
        assert abs((value(hi) - value(lo)) / (2 * step) - float(dx[r_, c])) < 1e-5


def test_ties_go_to_the_lowest_column_and_all_equal_rows():
    for V in (300, 2000, 4500):  # more equal columns than are collected, for one, one and two waves to a row
        r = Fn.token_logprobs(torch.zeros(2, V, device=DEV), top=64)
        assert torch.equal(r.top_index[0].cpu(), torch.arange(64))
    x = torch.zeros(4, 5000, dtype=torch.bfloat16, device=DEV)
    x[1, 4000:] = 3.0
    x[2, ::7] = 1.0
    x[3] = torch.randint(-2, 3, (5000,), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    r = Fn.token_logprobs(x, top=64)
    want = torch.sort(x.float().cpu(), dim=-1, descending=True, stable=True).indices[:, :64]
    assert torch.equal(r.top_index.cpu(), want)
    assert r.logprob is None and r.entropy is None
    assert abs(float(r.top_logprob[0, 0]) + math.log(5000)) < 1e-4


def test_sorted_rows_in_both_directions():
    """Every candidate in one thread's reach, or spread evenly: the selection has to hold for both."""
    up = torch.arange(20000, dtype=torch.float32).mul(1e-3)
    for n in (1000, 4000):  # (one and two waves to a row)
        for y in (up[:n], up[:n].flip(0)):
            r = Fn.token_logprobs(y[None].to(DEV), top=64)
            assert torch.equal(r.top_index[0].cpu(), torch.sort(y, descending=True, stable=True).indices[:64])
    blocks = torch.zeros(20000)
    blocks[256 * torch.arange(40) + 3] = torch.arange(40, dtype=torch.float32) + 1.0      # one residue class of 256
    dense = torch.zeros(20000)
    dense[8008:8072] = torch.arange(64, dtype=torch.float32) + 1.0                         # neighbours
    x = torch.stack([up, up.flip(0), blocks, dense]).to(DEV)
    r = Fn.token_logprobs(x, top=64)
    assert torch.equal(r.top_index.cpu(), torch.sort(x.cpu(), dim=-1, descending=True, stable=True).indices[:, :64])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_in_the_logits(dtype):
    """-inf columns (forbidden tokens), the type's lowest value, a forbidden target; rows of nothing but -inf, +inf and NaN come out NaN
    as log_softmax has it, and their neighbours are not touched."""
    x, g = _logits(8, 515, dtype, 3)
    x[0, 100:400] = -math.inf
    x[1, 7] = -math.inf
    x[2, 1:] = -math.inf
    x[3, 10:] = torch.finfo(dtype).min
    x[4] = -math.inf
    x[5, 3] = math.inf
    x[6, 3] = math.nan
    tokens = torch.tensor([0, 7, 0, 3, 5, 4, 4, 9])
    leaf = x.detach().requires_grad_()
    r = Fn.token_logprobs(leaf, tokens.to(DEV), top=3, entropy=True)
    (dx,) = torch.autograd.grad([r.logprob[[0, 2, 3, 7]].sum() + r.entropy[[0, 2, 3, 7]].sum()], leaf)
    xc = x.float().cpu()
    want = torch.log_softmax(xc.double(), -1)
    for i in (0, 2, 3, 7):
        ep = E * (8 * 20 + 515 / 64 + 64)
        assert abs(float(r.logprob[i]) - float(want[i, tokens[i]])) <= ep
        p = want[i].exp()
        h = float(-torch.where(p > 0, p * want[i], 0.0).sum())
        assert abs(float(r.entropy[i]) - h) <= ep * (2 * h + 2)
        assert torch.isfinite(dx[i]).all()
    assert not dx[0, 100:400].any()
    assert float(r.logprob[1]) == -math.inf and math.isfinite(float(r.entropy[1]))
    assert torch.equal(r.top_index[2].cpu(), torch.tensor([0, 1, 2]))
    for i in (4, 5, 6):
        assert math.isnan(float(r.logprob[i])) and math.isnan(float(r.entropy[i]))
    assert int(r.top_index.max()) < 515 and int(r.top_index.min()) >= -1


def test_a_token_outside_the_vocabulary_scores_nan():
    x, g = _logits(4, 33, torch.float32, 9)
    leaf = x.detach().requires_grad_()
    tokens = torch.tensor([33, -1, 5, 1 << 40], device=DEV)
    r = Fn.token_logprobs(leaf, tokens, entropy=True)
    assert torch.isnan(r.logprob).tolist() == [True, True, False, True] and torch.isfinite(r.entropy).all()
    (dx,) = torch.autograd.grad(r.logprob.sum(), leaf)
    assert torch.isfinite(dx[2]).all() and torch.isnan(dx[[0, 1, 3]]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_lead_dimensions_and_alignment(dtype):
    """Rows at any address and stride, a decoder's [B, U, V], a transposed view: the same numbers as from a contiguous copy."""
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(12, 1031, generator=g).to(dtype).to(DEV)
    for view in (wide[:, 1:1000], wide[:, 3:], wide[::2, 8:1000], wide[:, :999].unflatten(0, (3, 4)), wide[:, :999].unflatten(0, (3, 4)).transpose(0, 1)):
        tokens = torch.randint(0, view.shape[-1], view.shape[:-1], generator=g).to(DEV)
        a = Fn.token_logprobs(view, tokens, top=5, entropy=True)
        flat = view.contiguous().view(-1, view.shape[-1])
        b = Fn.token_logprobs(flat, tokens.reshape(-1), top=5, entropy=True)
        assert a.logprob.shape == view.shape[:-1] and a.top_index.shape == view.shape[:-1] + (5,)
        ep = _ep(flat.float().cpu(), 1.0)
        assert torch.equal(a.top_index.reshape(-1, 5), b.top_index)
        assert float((a.logprob.reshape(-1) - b.logprob).abs().max()) <= 2 * ep
        leaf = view.detach().requires_grad_()
        (dx,) = torch.autograd.grad(Fn.token_logprobs(leaf, tokens).logprob.sum(), leaf)
        assert dx.shape == view.shape and torch.isfinite(dx).all()


def test_an_empty_batch_and_partial_gradients():
    x = torch.empty(0, 10, device=DEV)
    r = Fn.token_logprobs(x, torch.empty(0, dtype=torch.int64, device=DEV), top=2, entropy=True)
    assert r.logprob.shape == (0,) and r.top_index.shape == (0, 2)
    x, g = _logits(6, 77, torch.float32, 4)
    tokens = torch.randint(0, 77, (6,), generator=g)
    for pick in ("logprob", "entropy", "top_logprob"):
        leaf = x.detach().requires_grad_()
        r = Fn.token_logprobs(leaf, tokens.to(DEV), top=4, entropy=True)
        o = getattr(r, pick)
        u = torch.randn(o.shape, generator=g)
        (dx,) = torch.autograd.grad(o, leaf, u.to(DEV))
        ups = [u if n == pick else None for n in ("logprob", "entropy", "top_logprob")]
        grad = _exact(x.cpu(), tokens, 4, 1.0, None, ups)[4]
        assert float((dx.cpu().double() - grad).abs().max()) <= 40 * _ep(x.cpu(), 1.0)  # |upstream| <= 4 in four terms, H <= log 77 < 5


def test_gradients_of_broadcast_logits_and_of_a_tensor_used_twice():
    """One row expanded to five, and the same logits scored for two sets of tokens: the gradients add up."""
    x, g = _logits(1, 50, torch.float32, 6, pad=False)
    tokens = torch.randint(0, 50, (5,), generator=g)
    up = torch.randn(5, generator=g)
    leaf = x.detach().requires_grad_()
    a = Fn.token_logprobs(leaf.expand(5, 50), tokens.to(DEV)).logprob
    b = Fn.token_logprobs(leaf, tokens[:1].to(DEV), entropy=True)
    (dx,) = torch.autograd.grad([a, b.logprob, b.entropy], leaf, [up.to(DEV), torch.ones(1, device=DEV), torch.ones(1, device=DEV)])
    xc = x.double().cpu().requires_grad_()
    lp = torch.log_softmax(xc, -1)
    (lp.expand(5, 50).gather(1, tokens[:, None])[:, 0] * up.double()).sum().add(lp[0, tokens[0]] - (lp.exp() * lp).sum()).backward()
    assert float((dx.cpu().double() - xc.grad).abs().max()) <= 60 * _ep(x.cpu(), 1.0)  # seven terms, |upstream| <= 3, H <= log 50 < 4


def test_logits_beyond_32_bit_offsets():
    """66 000 rows of 33 000: 2.2e9 elements; every row of zeros scores -log V, the last ones their own values, the gradient reaches them."""
    rows, V = 66000, 33000
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(3)
    x[-2:] = torch.randn(2, V, generator=g).bfloat16().to(DEV)
    tokens = torch.arange(rows, device=DEV) % V
    leaf = x.requires_grad_()
    r = Fn.token_logprobs(leaf, tokens, top=2)
    assert float((r.logprob[:-2] + math.log(V)).abs().max()) <= E * (V / 64 + 64)
    want = torch.log_softmax(x[-2:].detach().double().cpu(), -1)
    at = tokens[-2:].cpu()
    assert float((r.logprob[-2:].detach().cpu().double() - want.gather(1, at[:, None])[:, 0]).abs().max()) <= _ep(x[-2:].detach().float().cpu(), 1.0)
    assert torch.equal(r.top_index[-2:].cpu(), torch.sort(x[-2:].detach().float().cpu(), dim=-1, descending=True, stable=True).indices[:, :2])
    (dx,) = torch.autograd.grad(r.logprob[-1], leaf)
    assert not dx[:-1].any()
    exact = -want[1].exp()
    exact[at[1]] += 1
    assert bool(((dx[-1].cpu().double() - exact).abs() <= 2.0 ** -8 * exact.abs() + _ep(x[-1:].detach().float().cpu(), 1.0) * 2).all())


def test_a_second_derivative_is_refused():
    x, g = _logits(2, 9, torch.float32, 1)
    leaf = x.detach().requires_grad_()
    r = Fn.token_logprobs(leaf, torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(r.logprob.sum(), leaf, create_graph=True)


def test_two_runs_are_equal_and_a_graph_replays():
    x, g = _logits(300, 10000, torch.bfloat16, 8)
    tokens = torch.randint(0, 10000, (300,), generator=g).to(DEV)
    up = torch.randn(300, generator=g).to(DEV)

    def step():
        leaf = x.detach().requires_grad_()
        r = Fn.token_logprobs(leaf, tokens, top=6, entropy=True, ignore_index=1)
        (dx,) = torch.autograd.grad([r.logprob, r.entropy], leaf, [up, up])
        return r.logprob, r.entropy, r.top_logprob, r.top_index, dx

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        new, g2 = _logits(300, 10000, torch.bfloat16, 100 + seed)
        x.copy_(new)
        tokens.copy_(torch.randint(0, 10000, (300,), generator=g2))
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(held, step(), step()):
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num()) and torch.equal(b, c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [9, 1000, 40001])
def test_logits_far_from_zero(V, dtype):
    """A softmax does not change with an offset.  Rows of the type's lowest value alone, of numbers around 10^6 and -10^30, and with the type's
    largest value have the scores and gradients of the rows' differences: within ED = e (8 max |z - max z| + V / 64 + 64) as above, a
    difference below -200 (its p is 0 in fp32) counting as 200 where p multiplies it."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(6, V, generator=g) * 3
    x[1] = 1e6 + x[1] * 4
    x[2] = torch.finfo(dtype).min
    x[3] = -1e30 + x[3]
    x[4, V // 2] = torch.finfo(dtype).max
    x[5] = torch.where(torch.arange(V) % 3 == 1, x[5], torch.tensor(torch.finfo(dtype).min))
    x = x.to(dtype)
    tokens = torch.tensor([3, 5, 7, 1, V // 2, 4])
    ups = [torch.randn(6, generator=g), torch.randn(6, generator=g)]
    leaf = x.to(DEV).requires_grad_()
    r = Fn.token_logprobs(leaf, tokens.to(DEV), top=2, entropy=True)
    (dx,) = torch.autograd.grad([r.logprob, r.entropy], leaf, [u.to(DEV) for u in ups])
    lp, h, best, idx, grad, p, alllp = _exact(x.float(), tokens, 2, 1.0, None, ups)
    far = (alllp - alllp.amax(1, keepdim=True)).abs().clamp(max=200)
    ed = E * (8 * far.amax(1) + V / 64 + 64)
    assert torch.equal(r.top_index.cpu(), idx)
    assert bool(((r.logprob.cpu().double() - lp).abs() <= ed).all())
    assert bool(((r.top_logprob.cpu().double() - best).abs() <= ed[:, None]).all())
    assert bool(((r.entropy.cpu().double() - h).abs() <= ed * (2 * h + 2)).all())
    half = E if dtype == torch.float32 else 2.0 ** -8
    W, gh = ups[0].abs().double()[:, None], ups[1].abs().double()[:, None]
    size = alllp.abs().clamp(max=400)
    inner = W + gh * (size + h[:, None])
    # a p below the smallest normal number 2^-126 may be flushed: up to 2^-126 missing, times what p is multiplied with, and the product's own
    # flush (here p = 1.13e-38 < 2^-126 = 1.175e-38 and a factor of 43)
    bound = half * grad.abs() + p * inner * (ed[:, None] + 16 * E) + p * gh * ed[:, None] * (2 * h[:, None] + 3) + 2.0 ** -126 * (1 + inner)
    bound.scatter_add_(1, tokens[:, None], 4 * E * W)
    assert bool(((dx.cpu().double() - grad).abs() <= bound).all()), ((dx.cpu().double() - grad).abs() / bound).amax(1)
