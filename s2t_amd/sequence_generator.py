"""Autoregressive beam search on the HIP path.

Mirrors the contract of the reference's ``fairseq/sequence_generator.py`` (``SequenceGenerator.__init__`` :22-118,
``generate`` :176-189, ``_generate`` :191-614, ``finalize_hypos`` :650-786) with ``search.BeamSearch.step``
(``search.py:101-150``): same constructor arguments, same return value (per sentence a score-sorted list of dicts with
``tokens``, ``score``, ``attention``, ``alignment``, ``positional_scores``), same candidate rules —

  * step 0 expands the first beam only; later steps rank all (beam, token) pairs by cumulative log-probability;
  * pad and blank (``<s>``, index 0) are never selected, ``<unk>`` is penalised, ``</s>`` is forbidden before
    ``min_len`` and forced at ``max_len = min(int(a * src_len + b), max_decoder_positions - 1)``;
  * of the best ``2 * beam`` candidates an ``</s>`` among the first ``beam`` is finalised with
    ``score / (step + 1) ** len_penalty``; the first ``beam`` non-``</s>`` candidates continue;
  * a sentence stops once ``beam`` hypotheses are finished or ``step == max_len``.

The decoder runs incrementally (``TransformerDecoderScriptable`` with ``incremental_state``: per-layer key/value caches
in HBM, one query row per hypothesis, ``reorder_incremental_state`` after every step).  Finished sentences stay in the
batch (their rows are ignored) instead of being compacted away, which keeps every tensor shape static per step.
Joint CTC rescoring (``ctc_weight > 0``, reference :255-271 and :355-388): the reference pulls every hypothesis to the
host each step and scores it with ESPnet's numpy ``CTCPrefixScore`` through a dict keyed by the token string; here the
prefix states live in HBM ([rows, T', 2] fp32) and two launches of ``s2t_ctc_prefix_score`` per step score the
``int(1.5 * beam)`` candidates of every row and then advance the surviving rows' states — no per-token D2H.  The
reference scores all sentences against utterance 0 (``ctc_lprobs[0]``: a batch-size-1 path); this one scores each
sentence against its own frames, which is identical at batch size 1.
Greedy search with drafts (``draft="ctc"``, beam 1): the CTC head's transcript of the same encoder output is a draft of what the decoder is
about to say, and one pass of the decoder over a paged cache (s2t_amd/paged.py) verifies up to ``draft_len`` of its tokens at a time for every
sentence: the same hypotheses as beam 1 (up to rounding between equal scores) in fewer passes.  Behind a token where the decoder leaves
the draft it is not known whether the draft has one too few or a wrong one there, so the next pass carries both continuations as a tree.
Not built (reference options that the recipes' generation configs leave off): sampling / diverse / constrained search,
LM fusion, n-gram blocking, prefix tokens.
"""
import math
from typing import Dict, List, Optional

import torch

from . import functional as Fn
from . import kernels as K

CTC_SCORING_RATIO = 1.5  # sequence_generator.py:19


class SequenceGenerator:
    def __init__(self, models, tgt_dict, beam_size=1, max_len_a=0, max_len_b=200, min_len=1, normalize_scores=True,
                 len_penalty=1.0, unk_penalty=0.0, temperature=1.0, match_source_len=False, no_repeat_ngram_size=0,
                 search_strategy=None, eos=None, symbols_to_strip_from_output=None, lm_model=None, lm_weight=1.0,
                 ctc_weight=0.0, draft=None, draft_len=16):
        models = list(models) if isinstance(models, (list, tuple)) else [models]
        if len(models) != 1:
            raise NotImplementedError("model ensembles")
        if match_source_len or no_repeat_ngram_size or search_strategy is not None or lm_model is not None:
            raise NotImplementedError("only plain beam search is built on the HIP path (see module docstring)")
        self.model = models[0]
        self.tgt_dict = tgt_dict
        self.pad, self.unk = tgt_dict.pad(), tgt_dict.unk()
        self.eos = tgt_dict.eos() if eos is None else eos
        self.blank = tgt_dict.bos()
        self.vocab_size = len(tgt_dict)
        self.beam_size = min(beam_size, self.vocab_size - 1)  # sequence_generator.py:74-75
        self.max_len_a, self.max_len_b, self.min_len = max_len_a, max_len_b, min_len
        self.normalize_scores, self.len_penalty, self.unk_penalty = normalize_scores, len_penalty, unk_penalty
        self.temperature = temperature
        self.ctc_weight = float(ctc_weight)
        assert temperature > 0, "--temperature must be greater than 0"
        if draft not in (None, "ctc"):
            raise NotImplementedError("drafts from %r" % (draft,))
        if draft is not None and (self.beam_size != 1 or self.ctc_weight > 0 or draft_len < 1):
            raise ValueError("drafts verify greedy search: beam_size 1, no ctc_weight, draft_len >= 1")
        self.draft, self.draft_len = draft, int(draft_len)
        self.draft_passes = 0  # decoder passes of the last generate() with drafts

    @torch.no_grad()
    def generate(self, models, sample: Dict, drafts: Optional[List[List[int]]] = None, **kwargs) -> List[List[Dict]]:
        """``drafts`` (with ``draft``): token ids for each sentence, instead of the CTC head's."""
        if self.draft is not None:
            return self._generate_drafted(sample, drafts)
        return self._generate(sample)

    def _generate(self, sample):
        model = self.model
        model.eval()
        net_input = sample["net_input"]
        src_tokens, src_lengths = net_input["src_tokens"], net_input["src_lengths"]
        bsz, src_len = src_tokens.shape[:2]
        beam = self.beam_size
        dev = src_tokens.device
        max_len = min(int(self.max_len_a * src_len + self.max_len_b), model.decoder.max_positions() - 1)
        assert self.min_len <= max_len, "min_len cannot be larger than max_len, please adjust these!"

        enc = model.encoder(src_tokens, src_lengths)
        order = torch.arange(bsz, device=dev).view(-1, 1).repeat(1, beam).view(-1)
        ctc = None
        if self.ctc_weight > 0:
            ctc = self._ctc_prepare(enc, order, beam)
        enc = model.encoder.reorder_encoder_out(enc, order)

        tokens = torch.full((bsz * beam, max_len + 2), self.pad, dtype=torch.long, device=dev)
        tokens[:, 0] = self.eos
        scores = torch.zeros(bsz * beam, max_len + 1, dtype=torch.float32, device=dev)
        finalized: List[List[Dict]] = [[] for _ in range(bsz)]
        finished = [False] * bsz
        cand_size = 2 * beam
        bbsz_offsets = (torch.arange(bsz, device=dev) * beam).unsqueeze(1)
        cand_offsets = torch.arange(cand_size, device=dev)
        incremental_state: Dict = {}
        reorder: Optional[torch.Tensor] = None
        NEG = -math.inf

        for step in range(max_len + 1):
            if reorder is not None:
                model.decoder.reorder_incremental_state(incremental_state, reorder)
                enc = model.encoder.reorder_encoder_out(enc, reorder)
            logits, _ = model.decoder(tokens[:, :step + 1], encoder_out=enc, incremental_state=incremental_state)
            lprobs = torch.log_softmax(logits[:, -1, :].float() / self.temperature, dim=-1)
            if ctc is not None:
                self._ctc_rescore(ctc, lprobs, tokens, step)
            lprobs[lprobs != lprobs] = NEG
            lprobs[:, self.pad] = NEG
            lprobs[:, self.blank] = NEG
            lprobs[:, self.unk] -= self.unk_penalty
            if step >= max_len:
                lprobs[:, :self.eos] = NEG
                lprobs[:, self.eos + 1:] = NEG
            elif step < self.min_len:
                lprobs[:, self.eos] = NEG

            # ---- candidates (search.py:113-146)
            lp = lprobs.view(bsz, beam, self.vocab_size)
            if step == 0:
                lp = lp[:, :1, :]
            else:
                lp = lp + scores.view(bsz, beam, -1)[:, :, step - 1].unsqueeze(-1)
            flat = lp.reshape(bsz, -1)
            cand_scores, cand_flat = torch.topk(flat, k=min(cand_size, flat.size(1) - 1))
            cand_beams = torch.div(cand_flat, self.vocab_size, rounding_mode="trunc")
            cand_tokens = cand_flat.fmod(self.vocab_size)
            cand_bbsz = cand_beams + bbsz_offsets
            eos_mask = cand_tokens.eq(self.eos) & cand_scores.ne(NEG)

            # ---- finalise </s> candidates that sit in the first `beam` slots (host side: a handful of scalars)
            fin_mask = eos_mask[:, :beam].cpu()
            if bool(fin_mask.any()):
                cs, cb = cand_scores[:, :beam].cpu(), cand_bbsz[:, :beam].cpu()
                tok_cpu, sc_cpu = tokens[:, 1:step + 2].cpu(), scores[:, :step + 1].cpu()
                for sent in range(bsz):
                    if finished[sent]:
                        continue
                    for j in range(beam):
                        if fin_mask[sent, j] and len(finalized[sent]) < beam:
                            row = int(cb[sent, j])
                            hyp_tokens = tok_cpu[row].clone()
                            hyp_tokens[step] = self.eos
                            pos = sc_cpu[row].clone()
                            pos[step] = cs[sent, j]
                            pos[1:] = pos[1:] - pos[:-1].clone()
                            score = float(cs[sent, j])
                            if self.normalize_scores:
                                score /= (step + 1) ** self.len_penalty
                            finalized[sent].append({"tokens": hyp_tokens, "score": torch.tensor(score), "attention": None,
                                                    "alignment": torch.empty(0), "positional_scores": pos})
            for sent in range(bsz):
                if not finished[sent] and (len(finalized[sent]) == beam or step == max_len):
                    finished[sent] = True
            if all(finished) or step >= max_len:
                break

            # ---- the first `beam` candidates that are not </s> continue (sequence_generator.py:540-570)
            active_mask = eos_mask.to(cand_offsets.dtype) * cand_size + cand_offsets[:eos_mask.size(1)]
            _, active_hypos = torch.topk(active_mask, k=beam, dim=1, largest=False)
            active_bbsz = torch.gather(cand_bbsz, 1, active_hypos).view(-1)
            tokens[:, :step + 1] = tokens[:, :step + 1].index_select(0, active_bbsz)
            tokens.view(bsz, beam, -1)[:, :, step + 1] = torch.gather(cand_tokens, 1, active_hypos)
            if step > 0:
                scores[:, :step] = scores[:, :step].index_select(0, active_bbsz)
            scores.view(bsz, beam, -1)[:, :, step] = torch.gather(cand_scores, 1, active_hypos)
            reorder = active_bbsz
            if ctc is not None:
                self._ctc_advance(ctc, active_bbsz, tokens, step)

        for sent in range(bsz):
            finalized[sent].sort(key=lambda h: -float(h["score"]))
        return finalized

    # ---- greedy search with drafts ------------------------------------------------------------------------------------------
    def _generate_drafted(self, sample, drafts):
        from .s2t_transformer import CTCDecoder

        model = self.model
        model.eval()
        net_input = sample["net_input"]
        src_tokens = net_input["src_tokens"]
        bsz, src_len = src_tokens.shape[:2]
        dev = src_tokens.device
        max_len = min(int(self.max_len_a * src_len + self.max_len_b), model.decoder.max_positions() - 1)
        assert self.min_len <= max_len, "min_len cannot be larger than max_len, please adjust these!"
        enc = model.encoder(src_tokens, net_input["src_lengths"])
        if drafts is None:
            if not any(len(enc.get(k, [])) for k in ("ctc_logit", "xctc_logit")):
                raise ValueError("the model has no CTC head to draft with: pass drafts")
            drafts = [h[0]["tokens"].tolist() for h in CTCDecoder([model], dictionary=self.tgt_dict, blank_idx=self.blank).from_encoder(enc)]
        if len(drafts) != bsz:
            raise ValueError("%d drafts for %d sentences" % (len(drafts), bsz))
        drafts = [[t for t in d if 0 <= t < self.vocab_size and t not in (self.pad, self.blank, self.eos)] for d in drafts]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        state = model.decoder.paged_state(enc, max_len + 1 + 2 * self.draft_len)
        sents = [_DraftedSentence(d, self.eos) for d in drafts]
        self.draft_passes = 0
        while any(not s.done for s in sents):
            self.draft_passes += 1
            for b, s in enumerate(sents):
                s.plan(self.draft_len, max_len)
                if not s.done:  # (the pages of one that is done have been given back)
                    state.cache.reserve(b, s.kept + len(s.nodes))
            state.cache.sync()
            nodes = [n for s in sents for n in s.nodes]
            count = [len(s.nodes) for s in sents]
            most = max(count)
            cu = _offsets(count)
            state.lens.copy_(i32([s.kept + len(s.nodes) for s in sents]))
            tree = None
            if any(s.branches for s in sents):
                words = -(-most // 64)
                tree = torch.tensor([_words(n.sees, words) for n in nodes], dtype=torch.int64, device=dev)
            logits = model.decoder.extend(torch.tensor([n.token for n in nodes], device=dev),
                                          i32([s.kept + n.depth for s in sents for n in s.nodes]), state, i32(cu), most, tree)
            # five alternatives: of the best, at most pad, blank and a </s> that comes too early fall away, and <unk> may be penalised;
            # a bonus (a penalty below 0) may lift <unk> from any rank, so its own score comes with them
            r = _token_scores(logits, self.eos, min(5, self.vocab_size), self.temperature)
            of_eos, lps, ids = (x.tolist() for x in r)
            if self.unk_penalty < 0:
                of_unk = _token_scores(logits, self.unk, 0, self.temperature)[0].tolist()
                lps, ids = [x + [y] for x, y in zip(lps, of_unk)], [x + [self.unk] for x in ids]
            at = 0
            paths = []
            for s in sents:
                n = len(s.nodes)
                paths.append(s.walk([self._choice(s.step(i), max_len, of_eos[at + i], lps[at + i], ids[at + i]) for i in range(n)]) if n else [])
                at += n
            if any(p != list(range(len(p))) for p in paths):  # a path off the first branch: its places close ranks
                kept = [len(p) for p in paths]
                state.accept(i32([cu[b] + i for b, p in enumerate(paths) for i in p]), i32([s.kept for s in sents]), i32(_offsets(kept)), max(kept))
            for b, s in enumerate(sents):
                if s.done and state.cache.held[b]:
                    state.cache.release(b)
        out = []
        for s in sents:
            pos = torch.tensor(s.scores, dtype=torch.float32)
            score = float(pos.sum())
            if self.normalize_scores:
                score /= len(s.out) ** self.len_penalty
            out.append([{"tokens": torch.tensor(s.out), "score": torch.tensor(score), "attention": None, "alignment": torch.empty(0),
                         "positional_scores": pos}])
        return out

    def _choice(self, step, max_len, of_eos, lps, ids):
        """The greedy token of one row and its score, by the rules of ``_generate``."""
        if step >= max_len:
            return self.eos, of_eos
        best = (self.eos, -math.inf)
        for lp, t in zip(lps, ids):
            if t < 0 or t in (self.pad, self.blank) or (t == self.eos and step < self.min_len) or lp != lp:
                continue
            if t == self.unk:
                lp -= self.unk_penalty
            if lp > best[1]:
                best = (t, lp)
        return best

    # ---- joint CTC rescoring (reference :255-271, :355-388) -----------------------------------------------------------
    def _ctc_prepare(self, enc, order, beam):
        key = "xctc_logit" if len(enc.get("xctc_logit", [])) > 0 else "ctc_logit"  # :257-260
        logit = enc[key][0]  # (T', B, V), a view of the encoder's batch-major buffer
        Tn, B, V = logit.shape
        lp = torch.log_softmax(logit.transpose(0, 1).float(), dim=-1).reshape(B * Tn, V).contiguous()
        in_lens = (~enc["encoder_padding_mask"][0]).sum(1).to(torch.int32)
        sent = order.to(torch.int32).contiguous()
        R = sent.numel()
        state = torch.empty(R, Tn, 2, dtype=torch.float32, device=lp.device)
        K.ctc_prefix_init(lp, Tn, in_lens, sent, self.blank, state)
        return {"lp": lp, "T": Tn, "in_lens": in_lens, "sent": sent, "state": state,
                "prev": torch.zeros(R, dtype=torch.float32, device=lp.device),
                "row_len": in_lens.long().index_select(0, order), "k": min(V, int(beam * CTC_SCORING_RATIO))}

    def _ctc_rescore(self, ctc, lprobs, tokens, step):
        """lprobs[r, ids] <- (1 - w) * lprobs[r, ids] + w * (psi(prefix_r + ids) - psi(prefix_r)) for the ctc_beam best
        non-blank ids of every row, while step <= T' of the row's utterance (:355-382)."""
        masked = lprobs.clone()
        masked[:, self.blank] = -math.inf
        ids = torch.topk(masked, ctc["k"], dim=-1).indices.contiguous()
        psi = torch.empty(ids.shape, dtype=torch.float32, device=lprobs.device)
        K.ctc_prefix_score(ctc["lp"], ctc["T"], ctc["in_lens"], ctc["sent"], ctc["state"], tokens[:, step].contiguous(), step,
                           ids, self.blank, self.eos, psi)
        old = lprobs.gather(1, ids)
        new = (1.0 - self.ctc_weight) * old + self.ctc_weight * (psi - ctc["prev"].unsqueeze(1))
        live = (ctc["row_len"] >= step).unsqueeze(1)
        lprobs.scatter_(1, ids, torch.where(live, new, old))

    def _ctc_advance(self, ctc, parents, tokens, step):
        """The surviving rows' prefix states: parent state + the token just appended (tokens[:, step + 1]); ``tokens`` has
        already been re-ordered, so tokens[:, step] is the parent's last token."""
        parent_state = ctc["state"].index_select(0, parents)
        cand = tokens[:, step + 1].contiguous().view(-1, 1)
        psi = torch.empty(cand.shape, dtype=torch.float32, device=cand.device)
        new_state = torch.empty_like(parent_state).unsqueeze(1)
        K.ctc_prefix_score(ctc["lp"], ctc["T"], ctc["in_lens"], ctc["sent"], parent_state, tokens[:, step].contiguous(), step,
                           cand, self.blank, self.eos, psi, new_state)
        ctc["state"] = new_state.squeeze(1)
        ctc["prev"] = psi.view(-1)


def _token_scores(logits, token, top, temperature):
    """-> log probability of ``token`` in every row, the ``top`` best log probabilities and their ids."""
    r = Fn.token_logprobs(logits, torch.full((logits.shape[0],), token, device=logits.device), top=top, temperature=temperature)
    return r.logprob, r.top_logprob, r.top_index


def _offsets(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _words(bits, words):
    """A Python integer as ``words`` signed 64-bit words, the lowest first."""
    return [((bits >> (64 * w) & (1 << 64) - 1) ^ 1 << 63) - (1 << 63) for w in range(words)]


class _Node:
    """A token that the next pass feeds: ``at`` draft index behind it, ``sees`` bits of itself and its ancestors."""

    __slots__ = ("token", "depth", "at", "sees", "next")

    def __init__(self, token, depth, at, sees):
        self.token, self.depth, self.at, self.sees, self.next = token, depth, at, sees, {}


class _DraftedSentence:
    """One sentence of the search with drafts.  ``kept`` places are in the cache, ``out`` has been said; its last token (at first </s>) is fed
    next, as node 0, followed by what the draft has from ``at`` on and, where that may be one token late, from ``other`` on."""

    def __init__(self, draft, eos):
        self.draft, self.eos = draft, eos
        self.kept, self.out, self.scores = 0, [], []
        self.at, self.other, self.done = 0, None, False
        self.nodes, self.branches = [], False

    def step(self, i):
        return self.kept + self.nodes[i].depth

    def plan(self, draft_len, max_len):
        self.nodes, self.branches = [], False
        if self.done:
            return
        self.nodes.append(_Node(self.out[-1] if self.out else self.eos, 0, self.at, 1))
        most = min(draft_len, max_len - self.kept)
        for start in (self.at,) if self.other is None else (self.at, self.other):
            node = self.nodes[0]
            for j in range(start, min(start + most, len(self.draft))):
                i = node.next.get(self.draft[j])
                if i is None:
                    if node.next or node is not self.nodes[-1]:
                        self.branches = True
                    i = node.next[self.draft[j]] = len(self.nodes)
                    self.nodes.append(_Node(self.draft[j], node.depth + 1, j + 1, node.sees | 1 << i))
                node = self.nodes[i]

    def walk(self, choices):
        """Follows the decoder's choices from node 0 as far as the drafts agree -> the nodes that stay in the cache."""
        i, path = 0, []
        while True:
            path.append(i)
            token, score = choices[i]
            self.out.append(token)
            self.scores.append(score)
            if token == self.eos:
                self.done = True
                break
            if token not in self.nodes[i].next:
                break
            i = self.nodes[i].next[token]
        self.kept += len(path)
        at, d = self.nodes[i].at, self.draft
        if at < len(d) and d[at] == token:            # the draft goes on behind what this pass could take
            self.at, self.other = at + 1, None
        elif at + 1 < len(d) and d[at + 1] == token:  # the draft has a token too many
            self.at, self.other = at + 2, None
        else:                                         # a wrong one, or one too few
            self.at, self.other = min(at + 1, len(d)), at
        return path
