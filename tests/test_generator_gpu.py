"""Incremental decoder + beam search on the HIP path against (i) hypotheses generated by the
reference's SequenceGenerator (golden fixture) and (ii) its own teacher-forced decoder."""
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from s2t_amd import s2t_transformer as M  # noqa: E402
from s2t_amd.sequence_generator import SequenceGenerator  # noqa: E402
from tests.test_model_parity_gpu import args_from_cfg  # noqa: E402
from oracle import s2t_oracle as O  # noqa: E402

DEV = "cuda"


def test_beam_search_matches_reference_hypotheses(golden_dir):
    z = np.load(os.path.join(golden_dir, "beam_search_transformer.npz"))
    cfg = O.cfg_from_golden(z)
    vocab = z["w::decoder.embed_tokens.weight"].shape[0]
    args = args_from_cfg(cfg, vocab)
    task = M.FakeTask(vocab)
    model = M.S2TTransformerModel.build_model(args, task)
    model.load_state_dict({k[3:]: torch.from_numpy(z[k]) for k in z.files if k.startswith("w::")}, strict=True)
    model.prepare(torch.float32, DEV)
    gen = SequenceGenerator([model], task.target_dictionary, beam_size=int(z["gen::beam"]), max_len_a=0,
                            max_len_b=int(z["gen::max_len_b"]))
    sample = {"net_input": {"src_tokens": torch.from_numpy(z["in::src_tokens"]).to(DEV),
                            "src_lengths": torch.from_numpy(z["in::src_lengths"]).to(DEV)}}
    hyps = gen.generate([model], sample)
    assert [len(h) for h in hyps] == z["gen::n_hyps"].tolist()
    for b, hb in enumerate(hyps):
        for k, h in enumerate(hb):
            assert h["tokens"].tolist() == z["out::tokens_%d_%d" % (b, k)].tolist(), (b, k)
            assert abs(float(h["score"]) - float(z["out::score_%d_%d" % (b, k)])) < 1e-3
            np.testing.assert_allclose(h["positional_scores"].numpy(), z["out::pos_scores_%d_%d" % (b, k)], atol=2e-3)


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-3), (torch.bfloat16, 4e-2)])
def test_incremental_steps_equal_teacher_forced_decoder(dtype, tol):
    """Every step of the cached decoder reproduces the corresponding position of the full (teacher-forced) decoder;
    64-wide heads in bf16 take the fused attention kernel with one query row."""
    torch.manual_seed(3)
    V = 47
    args = M.recipe_args(conformer=False, encoder_embed_dim=128, encoder_ffn_embed_dim=256, encoder_layers=2,
                         decoder_layers=2, decoder_embed_dim=128, decoder_ffn_embed_dim=256, encoder_attention_heads=2,
                         decoder_attention_heads=2, subsampling_filter=96, vocab_size=V)
    model = M.S2TTransformerModel.build_model(args, M.FakeTask(V)).prepare(dtype, DEV)
    model.eval()
    g = torch.Generator().manual_seed(1)
    B, T, U = 3, 120, 19
    lens = torch.tensor([120, 100, 77])
    src = torch.randn(B, T, 80, generator=g)
    for b in range(B):
        src[b, lens[b]:] = 0
    prev = torch.randint(4, V, (B, U), generator=g)
    prev[:, 0] = 2
    with torch.no_grad():
        enc = model.encoder(src.to(DEV), lens.to(DEV))
        full, _ = model.decoder(prev.to(DEV), encoder_out=enc)
        state = {}
        for t in range(U):
            step, _ = model.decoder(prev[:, :t + 1].to(DEV), encoder_out=enc, incremental_state=state)
            ref = full[:, t].float()
            err = (step[:, 0].float() - ref).abs().max() / ref.abs().max()
            assert float(err) < tol, (t, float(err))
            if t == 7:  # reorder mid-way: the caches must follow the permutation
                perm = torch.tensor([2, 0, 1], device=DEV)
                model.decoder.reorder_incremental_state(state, perm)
                enc = model.encoder.reorder_encoder_out(enc, perm)
                prev = prev[perm.cpu()]
                full = full[perm]


def test_ctc_prefix_score_kernel_matches_scorer():
    """s2t_ctc_prefix_init/_score against the oracle's restatement of the ESPnet scorer: chains of prefixes (repeated
    labels, </s> and blank among the candidates), ragged utterance lengths, states and scores."""
    from s2t_amd import kernels as K
    g = torch.Generator().manual_seed(9)
    B, T, V, blank, eos, beam, Kc = 3, 37, 13, 0, 2, 2, 5
    lens = torch.tensor([37, 29, 6], dtype=torch.int32)
    lp = torch.log_softmax(torch.randn(B, T, V, generator=g) * 2, -1)
    sent = torch.arange(B, dtype=torch.int32).repeat_interleave(beam)
    R = B * beam
    lpd = lp.reshape(B * T, V).to(DEV)
    state = torch.empty(R, T, 2, device=DEV)
    K.ctc_prefix_init(lpd, T, lens.to(DEV), sent.to(DEV), blank, state)
    scorers = [O.CTCPrefixScore(lp[b, :lens[b]].numpy(), blank, eos) for b in range(B)]
    ref_state = [scorers[int(sent[r])].initial_state() for r in range(R)]
    for r in range(R):
        n = int(lens[sent[r]])
        np.testing.assert_allclose(state[r, :n].cpu().numpy(), ref_state[r], rtol=1e-5, atol=1e-4)
    prefixes = [[eos] for _ in range(R)]
    for step in range(8):  # runs past the 6-frame utterance: rows with more labels than frames report logzero
        cand = torch.randint(3, V, (R, Kc), generator=g)
        cand[:, 0] = eos
        cand[:, 1] = blank
        if step > 0:
            cand[:, 2] = torch.tensor([p[-1] for p in prefixes])  # repeat of the last label
        last = torch.tensor([p[-1] for p in prefixes])
        psi = torch.empty(R, Kc, device=DEV)
        new = torch.empty(R, Kc, T, 2, device=DEV)
        K.ctc_prefix_score(lpd, T, lens.to(DEV), sent.to(DEV), state, last.to(DEV), step, cand.to(DEV), blank, eos, psi, new)
        pick = torch.randint(2, Kc, (R,), generator=g)
        nxt = []
        for r in range(R):
            n = int(lens[sent[r]])
            if step > n:
                assert (psi[r].cpu() == -1e10).all()
                nxt.append(ref_state[r])
                continue
            rp, rs = scorers[int(sent[r])](prefixes[r], cand[r].numpy(), ref_state[r])
            np.testing.assert_allclose(psi[r].cpu().numpy(), rp, rtol=1e-4, atol=2e-3)
            lo = max(step - 1, 0)
            np.testing.assert_allclose(new[r, :, lo:n].cpu().numpy(), rs[:, lo:], rtol=1e-4, atol=2e-3)
            nxt.append(rs[int(pick[r])])
        ref_state = nxt
        state = new[torch.arange(R), pick.to(DEV)].contiguous()
        prefixes = [p + [int(cand[r, pick[r]])] for r, p in enumerate(prefixes)]


def test_joint_ctc_beam_search_matches_oracle(golden_dir):
    """ctc_weight > 0: hypotheses of the on-device joint search against the oracle's host-side restatement (the reference's
    own joint path cannot run here: it needs ESPnet and hard-codes ``.to(device="cuda")``, sequence_generator.py:379-381)."""
    z = np.load(os.path.join(golden_dir, "beam_search_transformer.npz"))
    cfg = O.cfg_from_golden(z)
    vocab = z["w::decoder.embed_tokens.weight"].shape[0]
    task = M.FakeTask(vocab)
    model = M.S2TTransformerModel.build_model(args_from_cfg(cfg, vocab), task)
    model.load_state_dict({k[3:]: torch.from_numpy(z[k]) for k in z.files if k.startswith("w::")}, strict=True)
    model.prepare(torch.float32, DEV)
    beam, mlb = int(z["gen::beam"]), int(z["gen::max_len_b"])
    src, lens = torch.from_numpy(z["in::src_tokens"]), torch.from_numpy(z["in::src_lengths"])
    gen = SequenceGenerator([model], task.target_dictionary, beam_size=beam, max_len_a=0, max_len_b=mlb, ctc_weight=0.3)
    hyps = gen.generate([model], {"net_input": {"src_tokens": src.to(DEV), "src_lengths": lens.to(DEV)}})
    ref = O.beam_search(src, lens, O.weights_from_golden(z), cfg, beam=beam, max_len_b=mlb, ctc_weight=0.3)
    plain = O.beam_search(src[:1], lens[:1], O.weights_from_golden(z), cfg, beam=beam, max_len_b=mlb)
    assert [h["score"] for h in ref[0]] != [h["score"] for h in plain[0]]
    assert [len(h) for h in hyps] == [len(h) for h in ref]
    for b, hb in enumerate(hyps):
        for k, h in enumerate(hb):
            assert h["tokens"].tolist() == ref[b][k]["tokens"], (b, k)
            assert abs(float(h["score"]) - ref[b][k]["score"]) < 2e-3


def _golden_generator(golden_dir, **kw):
    z = np.load(os.path.join(golden_dir, "beam_search_transformer.npz"))
    cfg = O.cfg_from_golden(z)
    vocab = z["w::decoder.embed_tokens.weight"].shape[0]
    task = M.FakeTask(vocab)
    model = M.S2TTransformerModel.build_model(args_from_cfg(cfg, vocab), task)
    model.load_state_dict({k[3:]: torch.from_numpy(z[k]) for k in z.files if k.startswith("w::")}, strict=True)
    model.prepare(torch.float32, DEV)
    sample = {"net_input": {"src_tokens": torch.from_numpy(z["in::src_tokens"]).to(DEV), "src_lengths": torch.from_numpy(z["in::src_lengths"]).to(DEV)}}
    gen = lambda **k: SequenceGenerator([model], task.target_dictionary, max_len_a=0, max_len_b=int(z["gen::max_len_b"]), **kw, **k)  # noqa: E731
    return gen, sample, model


def _same_hypotheses(a, b, tol=1e-3):
    for x, y in zip(a, b):
        assert x[0]["tokens"].tolist() == y[0]["tokens"].tolist()
        assert abs(float(x[0]["score"]) - float(y[0]["score"])) < tol
        np.testing.assert_allclose(x[0]["positional_scores"].numpy(), y[0]["positional_scores"].numpy(), atol=2 * tol)


@pytest.mark.parametrize("kw", [{}, {"min_len": 6, "unk_penalty": 0.5}, {"temperature": 1.7, "len_penalty": 0.6}, {"normalize_scores": False}])
def test_greedy_search_with_drafts_equals_beam_one(golden_dir, kw):
    """Whatever the drafts — the CTC head's, none, the hypotheses themselves, hypotheses with tokens replaced, dropped and put in, other
    sentences' — the hypotheses are those of beam 1; right drafts take a fraction of the passes."""
    gen, sample, model = _golden_generator(golden_dir, **kw)
    want = gen(beam_size=1).generate([model], sample)
    right = [h[0]["tokens"].tolist()[:-1] for h in want]
    longest = max(len(h) for h in right) + 1
    drafted = gen(beam_size=1, draft="ctc", draft_len=5)
    _same_hypotheses(drafted.generate([model], sample), want)
    assert drafted.draft_passes <= longest
    edits = [[d[0] + 1] + d[1:2] + d[3:6] + [9] + d[6:] if len(d) > 6 else [7] + d for d in right]
    for drafts in ([[] for _ in right], right, edits, [list(reversed(d)) for d in right], right[1:] + right[:1], [d + [5] * 70 for d in edits]):
        for n in (1, 5, 40):
            g = gen(beam_size=1, draft="ctc", draft_len=n)
            _same_hypotheses(g.generate([model], sample, drafts=drafts), want)
            assert g.draft_passes <= longest
            if drafts is right and n == 40:
                assert g.draft_passes == 1 + (longest > 41)


@pytest.mark.parametrize("bonus", [0.5, 2.0, 4.0, 30.0])
def test_greedy_search_with_drafts_and_a_bonus_for_unk_equals_beam_one(golden_dir, bonus):
    """A negative penalty lifts <unk> from any rank, below the alternatives that a pass fetches too."""
    gen, sample, model = _golden_generator(golden_dir, unk_penalty=-bonus)
    want = gen(beam_size=1).generate([model], sample)
    right = [h[0]["tokens"].tolist()[:-1] for h in want]
    assert bonus < 30 or all(t == model.decoder.dictionary.unk() for h in right for t in h)
    for drafts in (right, [d[:1] + d[2:] for d in right], [[] for _ in right]):
        for n in (1, 5):
            _same_hypotheses(gen(beam_size=1, draft="ctc", draft_len=n).generate([model], sample, drafts=drafts), want)


def test_drafts_are_refused_where_they_cannot_verify(golden_dir):
    gen, sample, model = _golden_generator(golden_dir)
    with pytest.raises(ValueError, match="beam_size 1"):
        gen(beam_size=2, draft="ctc")
    with pytest.raises(ValueError, match="beam_size 1"):
        gen(beam_size=1, draft="ctc", ctc_weight=0.3)
    with pytest.raises(NotImplementedError):
        gen(beam_size=1, draft="lm")
    with pytest.raises(ValueError, match="drafts for"):
        gen(beam_size=1, draft="ctc").generate([model], sample, drafts=[[5]])


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-3), (torch.bfloat16, 4e-2)])
def test_extended_decoder_equals_teacher_forced_decoder(dtype, tol):
    """Passes of several tokens at a time over the paged cache — ragged, some sentences bringing none, a tree of drafts whose accepted path
    closes ranks — reproduce the positions of the full decoder (the bounds of the one-token test above)."""
    torch.manual_seed(3)
    V = 47
    args = M.recipe_args(conformer=False, encoder_embed_dim=128, encoder_ffn_embed_dim=256, encoder_layers=2, decoder_layers=2,
                         decoder_embed_dim=128, decoder_ffn_embed_dim=256, encoder_attention_heads=2, decoder_attention_heads=2,
                         subsampling_filter=96, vocab_size=V)
    model = M.S2TTransformerModel.build_model(args, M.FakeTask(V)).prepare(dtype, DEV)
    model.eval()
    g = torch.Generator().manual_seed(1)
    B, T, U = 3, 120, 19
    lens = torch.tensor([120, 100, 77])
    src = torch.randn(B, T, 80, generator=g)
    for b in range(B):
        src[b, lens[b]:] = 0
    prev = torch.randint(4, V, (B, U), generator=g)
    prev[:, 0] = 2
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    with torch.no_grad():
        enc = model.encoder(src.to(DEV), lens.to(DEV))
        full, _ = model.decoder(prev.to(DEV), encoder_out=enc)
        full = full.float()
        state = model.decoder.paged_state(enc, U + 8, page_size=8)
        for b in range(B):
            state.cache.reserve(b, U + 8)
        state.cache.sync()
        done = [0] * B

        def go(count, tokens, depths, tree=None):
            cu = [0] + list(np.cumsum(count))
            state.lens.copy_(i32([d + n for d, n in zip(done, count)]))
            pos = [done[b] + depths[cu[b] + i] for b in range(B) for i in range(count[b])]
            return cu, model.decoder.extend(torch.tensor(tokens, device=DEV), i32(pos), state, i32(cu), max(count), tree).float()

        def near(row, b, t):
            assert float((row - full[b, t]).abs().max() / full[b, t].abs().max()) < tol, (b, t)

        for count in ([4, 1, 0], [0, 3, 7], [1, 1, 1]):
            cu, logits = go(count, [int(prev[b, done[b] + i]) for b in range(B) for i in range(count[b])], [i for n in count for i in range(n)])
            for b in range(B):
                for i in range(count[b]):
                    near(logits[cu[b] + i], b, done[b] + i)
                done[b] += count[b]
        # a tree: node 0 the right token, node 1 a wrong child, node 2 the right child, node 3 a wrong child of 1, node 4 the right one of 2
        count, depths, sees = [5] * B, [0, 1, 1, 2, 2] * B, [1, 3, 5, 11, 21] * B
        tokens = [t for b in range(B) for t in (int(prev[b, done[b]]), 6, int(prev[b, done[b] + 1]), 7, int(prev[b, done[b] + 2]))]
        cu, logits = go(count, tokens, depths, torch.tensor(sees, device=DEV).view(-1, 1))
        for b in range(B):
            for node, t in ((0, 0), (2, 1), (4, 2)):
                near(logits[cu[b] + node], b, done[b] + t)
        done = [d + 3 for d in done]
        state.accept(i32([cu[b] + i for b in range(B) for i in (0, 2, 4)]), i32(done), i32([0, 3, 6, 9]), 3)
        count = [U - d for d in done]
        cu, logits = go(count, [int(prev[b, done[b] + i]) for b in range(B) for i in range(count[b])], [i for n in count for i in range(n)])
        for b in range(B):
            for i in range(count[b]):
                near(logits[cu[b] + i], b, done[b] + i)
