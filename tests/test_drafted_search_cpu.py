"""Greedy search with drafts against beam 1, both on a decoder that is a table: a sequence's next logits depend on its tokens alone, the
passes over the paged cache read them from what the cache, the drafts and the tree's words say.  No kernels: token scores in plain torch."""
import random
import types

import pytest
import torch

from s2t_amd import functional as Fn
from s2t_amd import paged
from s2t_amd.s2t_transformer import _DictLike
from s2t_amd.sequence_generator import SequenceGenerator


class _Decoder:
    """Logits of sentence b behind tokens ``said``: of a generator seeded by them, so that no two rows agree by chance."""

    def __init__(self, vocab, row, pages=None):
        self.vocab, self.row, self.pages, self.states, self.synced = vocab, row, pages, [], []

    def max_positions(self):
        return 64

    def logits(self, b, said):
        return self.row(torch.Generator().manual_seed(hash((b, tuple(said))) % (1 << 62)), b, said)

    def reorder_incremental_state(self, state, order):
        pass

    def __call__(self, tokens, encoder_out, incremental_state):
        return torch.stack([self.logits(b, t) for b, t in enumerate(tokens.tolist())])[:, None], None

    def paged_state(self, enc, places):
        state = types.SimpleNamespace(lens=torch.zeros(enc, dtype=torch.int32), places=[{} for _ in range(enc)])
        n = -(-places // 4)
        state.cache = paged.PagedKVCache(1, enc, self.pages or enc * n, n, 1, 16, torch.float32, "cpu", page_size=4)
        plain = state.cache.sync

        def sync():
            self.synced.append((state.cache.dirty, [len(h) for h in state.cache.held]))
            plain()
        state.cache.sync = sync

        def accept(rows, lens, cu, most):
            for b, place in enumerate(state.places):
                n = int(cu[b + 1] - cu[b])
                for i in range(n):
                    place[int(lens[b]) - n + i] = state.last[int(rows[int(cu[b]) + i])]
        state.accept = accept
        return state

    def extend(self, tokens, positions, state, cu, most, tree):
        state.last, out = tokens.tolist(), []
        for b, place in enumerate(state.places):
            first, n = int(cu[b]), int(cu[b + 1] - cu[b])
            at = int(state.lens[b]) - n
            assert n == 0 or len(state.cache.held[b]) * 4 >= at + n
            prefix = [place[p] for p in range(at)]
            for i in range(n):
                sees = [j for j in range(n) if (j <= i if tree is None else int(tree[first + i, j // 64]) >> (j % 64) & 1)]
                assert int(positions[first + i]) == at + len(sees) - 1
                out.append(self.logits(b, prefix + [state.last[first + j] for j in sees]))
            for i in range(n):
                place[at + i] = state.last[first + i]
        return torch.stack(out)


class _Encoder:
    def __call__(self, src, lengths):
        return src.shape[0]

    def reorder_encoder_out(self, enc, order):
        return enc


def _model(decoder):
    return types.SimpleNamespace(decoder=decoder, encoder=_Encoder(), eval=lambda: None)


@pytest.fixture(autouse=True)
def plain_scores(monkeypatch):
    def scores(logits, tokens=None, top=0, entropy=False, temperature=1.0, ignore_index=None):
        lp = torch.log_softmax(logits.float() / temperature, -1)
        best = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :top]
        return Fn.TokenScores(lp.gather(1, tokens[:, None])[:, 0], None, lp.gather(1, best) if top else None, best if top else None)
    monkeypatch.setattr(Fn, "token_logprobs", scores)


def _sample(n, frames=8):
    return {"net_input": {"src_tokens": torch.zeros(n, frames, 1), "src_lengths": torch.full((n,), frames)}}


VOCAB, EOS, UNK = 20, 2, 3


def _random_row(end):
    """Standard normal logits; </s> gains with the length, so that sentences end at different steps."""
    def row(g, b, said):
        x = torch.randn(VOCAB, generator=g)
        x[EOS] += (len(said) - end[b]) * 0.4
        return x
    return row


def _same(got, want):
    for x, y in zip(got, want):
        assert x[0]["tokens"].tolist() == y[0]["tokens"].tolist()
        assert abs(float(x[0]["score"]) - float(y[0]["score"])) < 1e-4  # (beam 1 sums its scores, 31 of up to 50, in another order: 2^-24 of 1550 each time, over the length)


@pytest.mark.parametrize("kw", [{}, {"unk_penalty": -0.5}, {"unk_penalty": -1.5}, {"unk_penalty": -2.5, "temperature": 1.7, "min_len": 4}, {"unk_penalty": 1.5},
                                {"unk_penalty": -50.0}])
def test_hypotheses_are_those_of_beam_one_whatever_unk_costs(kw):
    """A bonus lifts <unk> from any rank, also from below the alternatives that are fetched."""
    end = [3, 9, 14, 25]
    decoder = _Decoder(VOCAB, _random_row(end))
    model, task = _model(decoder), _DictLike(VOCAB)
    make = lambda **k: SequenceGenerator([model], task, beam_size=1, max_len_b=30, **kw, **k)  # noqa: E731
    want = make().generate([model], _sample(4))
    right = [h[0]["tokens"].tolist()[:-1] for h in want]
    if -50 < kw.get("unk_penalty", 0) < 0:  # the case that this is about is among them
        ranks = [int((decoder.logits(b, [EOS] + r[:i]) > decoder.logits(b, [EOS] + r[:i])[UNK]).sum()) for b, r in enumerate(right) for i, t in enumerate(r) if t == UNK]
        assert kw["unk_penalty"] > -1 or max(ranks) >= 5, ranks
    rng = random.Random(5)
    wrong = [[rng.randint(3, VOCAB - 1) if rng.random() < 0.2 else t for t in r] for r in right]
    for drafts in (right, wrong, [[] for _ in right], [r[:2] + r[3:] for r in right], right[1:] + right[:1]):
        for n in (1, 4, 30):
            _same(make(draft="ctc", draft_len=n).generate([model], _sample(4), drafts=drafts), want)


@pytest.mark.parametrize("kw", [{}, {"draft_len": 3}])
def test_sentences_that_are_done_hold_no_pages(kw):
    """From the pass behind its last one on a finished sentence holds none and does not have the table copied; a pool too small for
    all sentences at their full lengths serves them if the long ones outlive the short ones."""
    end = [2, 4, 6, 28]
    decoder = _Decoder(VOCAB, _random_row(end))
    model, task = _model(decoder), _DictLike(VOCAB)
    want = SequenceGenerator([model], task, beam_size=1, max_len_b=30).generate([model], _sample(4))
    lengths = [len(h[0]["tokens"]) for h in want]
    assert sorted(lengths)[-2] + 12 < max(lengths)
    make = lambda: SequenceGenerator([model], task, beam_size=1, max_len_b=30, draft="ctc", **kw)  # noqa: E731 (of the model at hand)
    _same(make().generate([model], _sample(4), drafts=[[]] * 4), want)   # a token to a pass
    assert len(decoder.synced) == max(lengths)
    for step, (dirty, held) in enumerate(decoder.synced):  # in the pass that feeds token `step` of each
        assert [h > 0 for h in held] == [step < n for n in lengths], (step, held, lengths)
        # a sentence gave its pages back at the end of the pass before, or one has come to a new page
        assert dirty == (step in lengths or any(step % 4 == 0 and step < n for n in lengths)), step
    assert any(not dirty for dirty, _ in decoder.synced[sorted(lengths)[-2] + 1:])
    pages = -(-max(lengths) // 4) + 3                      # the longest alone, and three more
    assert max(sum(-(-(step + 1) // 4) for n in lengths if step < n) for step in range(max(lengths))) <= pages < sum(-(-n // 4) for n in lengths)
    model = _model(_Decoder(VOCAB, _random_row(end), pages=pages))
    _same(make().generate([model], _sample(4), drafts=[[]] * 4), want)
