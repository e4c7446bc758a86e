"""A pre-norm decoder language model built on the FirstPassageAttention layer.

The training-step workload of the build's LM measurements: token embedding, `layers` blocks of
[LayerNorm -> FirstPassageAttention -> residual, LayerNorm -> GELU MLP -> residual], a final
LayerNorm and an output head tied to the embedding.  The reference ships the attention layer
(kernel.py:512-530) but no model around it; this one has the usual GPT-2-small shape (d_model 768,
12 heads, MLP 3072) so that a step exercises the layer at the size it is meant for.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import FirstPassageAttention, verify_drafts
from .cache import PAGE


class DecoderBlock(nn.Module):
    def __init__(self, d_model, n_heads, d_mlp, impl=None):
        super().__init__()
        self.ln1 = nn.LayerNorm(d_model)
        self.attn = FirstPassageAttention(d_model, n_heads, impl=impl)
        self.ln2 = nn.LayerNorm(d_model)
        self.fc1 = nn.Linear(d_model, d_mlp)
        self.fc2 = nn.Linear(d_mlp, d_model)

    def mlp(self, x):
        return x + self.fc2(F.gelu(self.fc1(self.ln2(x))))

    def forward(self, x):
        return self.mlp(x + self.attn(self.ln1(x)))


class DecodeState:
    """What a model keeps of B sequences while it answers: a cache and the last W of each layer, one table and the lengths
    of them all, and, where the sequences are samples of one prompt, that prompt as a shared prefix (pages, length)."""

    def __init__(self, caches, w, table, lengths, prefix=None):
        self.caches, self.w, self.table, self.lengths, self.prefix = caches, w, table, lengths, prefix
        self._new = None  # W of the positions of the last extend, per layer

    def keep(self, n):
        """Ends an extend of which n[b] (int32) positions stay (drafts behind them were rejected)."""
        at = (n.long() - 1).clamp(min=0).view(-1, 1, 1)
        self.w = [torch.where((n > 0).unsqueeze(1), new.gather(2, at.expand(-1, new.shape[1], 1)).squeeze(2), old)
                  for old, new in zip(self.w, self._new)]
        self.lengths = self.lengths + n
        self._new = None


class FPADecoder(nn.Module):
    """tokens (B, T) int64 -> logits (B, T, vocab)."""

    def __init__(self, vocab=32000, d_model=768, n_heads=12, layers=12, d_mlp=3072, impl=None):
        super().__init__()
        self.vocab = vocab
        self.emb = nn.Embedding(vocab, d_model)
        self.blocks = nn.ModuleList(DecoderBlock(d_model, n_heads, d_mlp, impl) for _ in range(layers))
        self.ln = nn.LayerNorm(d_model)
        self.head = nn.Linear(d_model, vocab, bias=False)
        self.head.weight = self.emb.weight
        nn.init.normal_(self.emb.weight, std=0.02)

    def forward(self, tokens):
        x = self.emb(tokens)
        for blk in self.blocks:
            x = blk(x)
        return self.head(self.ln(x))

    def loss(self, tokens):
        """Next-token cross entropy of tokens (B, T + 1): inputs tokens[:, :-1], targets tokens[:, 1:].

        The log-softmax reads the (fp16 under autocast) logits and works and writes in fp32 itself, so
        no fp32 copy of the logits is made first (the same values as cross_entropy on logits.float());
        autocast is off around it, since it would otherwise make that copy."""
        logits = self(tokens[:, :-1])
        with torch.autocast(device_type=logits.device.type, enabled=False):
            logp = torch.log_softmax(logits.reshape(-1, self.vocab), -1, dtype=torch.float32)
            return F.nll_loss(logp, tokens[:, 1:].reshape(-1))

    @torch.no_grad()
    def start(self, tokens, room, counts=None, samples=None, store=None):
        """Reads prompts (B, T), sequence b of counts[b] tokens (all T without counts), and returns (logits (B, vocab) behind the
        last of each, DecodeState with room for `room` more positions a sequence; beyond that logits are NaN).  samples: continue
        the one prompt that often; its positions are then kept once, and counts is None.  store: the caches' type,
        torch.float8_e4m3fn for 8 bits (None: the activations')."""
        B, T = tokens.shape
        dev = tokens.device
        if B < 1 or T < 1 or room < 0:
            raise ValueError("start needs a prompt of at least one token and room >= 0")
        if samples is not None and (B != 1 or samples < 1 or counts is not None):
            raise ValueError("samples, one or more, are taken of one whole prompt")
        if counts is None:
            counts = torch.full((B,), T, dtype=torch.int32, device=dev)
        else:
            counts = counts.to(torch.int32)
            if counts.shape != (B,) or bool(((counts < 1) | (counts > T)).any()):
                raise ValueError("counts must be (B,), each between 1 and T")
        first = -(-(T if samples is not None else T + room) // PAGE)
        own = max(-(-room // PAGE), 1) if samples is not None else 0
        table = torch.arange(B * first + (samples or 0) * own, dtype=torch.int32, device=dev)
        prompts, own_table = table[:B * first].view(B, first), table[B * first:].view(-1, own) if samples is not None else None
        x = self.emb(tokens)
        caches, ws = [], []
        for blk in self.blocks:
            caches.append(blk.attn.new_cache(table.numel(), x, store))
            y, w = blk.attn.prompt(blk.ln1(x), caches[-1], prompts, counts)
            x = blk.mlp(x + y)
            ws.append(w)
        logits = self.head(self.ln(x[torch.arange(B, device=dev), counts.long() - 1]))
        if samples is None:
            return logits, DecodeState(caches, ws, prompts, counts)
        return logits.expand(samples, -1), DecodeState(caches, [w.expand(samples, -1) for w in ws], own_table,
                                                       torch.zeros(samples, dtype=torch.int32, device=dev), (prompts[0], T))

    @torch.no_grad()
    def extend(self, state, tokens, keep=True):
        """Logits (B, N, vocab) behind each of N new tokens (B, N).  keep=False: state.keep(n) follows, with how many stay."""
        x = self.emb(tokens)
        new = []
        for blk, cache, w in zip(self.blocks, state.caches, state.w):
            y, w = blk.attn.extend(blk.ln1(x), cache, state.table, state.lengths, w, state.prefix)
            x = blk.mlp(x + y)
            new.append(w)
        state._new = new
        if keep:
            state.keep(torch.full_like(state.lengths, tokens.shape[1]))
        return self.head(self.ln(x))


def _sample(probs, u):
    """One token (B, 1) a sequence from probs (B, vocab) and uniforms u (B,)."""
    B = probs.shape[0]
    none = torch.empty(B, 0, dtype=torch.int64, device=probs.device)
    return verify_drafts(probs.unsqueeze(1), None, none, none.float(), u)[1]


@torch.no_grad()
def generate(model, tokens, steps, counts=None, samples=None, draft=None, drafts=4, temperature=1.0, generator=None, store=None):
    """tokens (B, steps) int64 sampled behind the prompts `tokens` (see FPADecoder.start).  draft: a smaller model that proposes
    `drafts` tokens at a time, of which `model` accepts what keeps its own distribution (verify_drafts).  Logits that are no
    distribution (NaN) give -1, after which the sequence goes on as if behind token 0."""
    if steps < 1 or not temperature > 0 or (draft is not None and drafts < 1):
        raise ValueError("generate needs steps >= 1, temperature > 0 and drafts >= 1")
    dev = tokens.device

    def uniform(*shape):
        return torch.rand(*shape, generator=generator, device=dev)

    def probs(logits):
        return torch.softmax(logits.float() / temperature, -1)
    room = steps + (drafts + 1 if draft is not None else 0)
    logits, state = model.start(tokens, room, counts, samples, store)
    B = logits.shape[0]
    last = _sample(probs(logits), uniform(B))
    if draft is None:
        out = [last]
        for _ in range(steps - 1):
            out.append(_sample(probs(model.extend(state, out[-1].clamp(min=0))[:, 0]), uniform(B)))
        return torch.cat(out, 1)
    _, guess = draft.start(tokens, room, counts, samples, store)
    out = torch.full((B, steps + drafts + 1), -1, dtype=torch.int64, device=dev)
    out[:, :1] = last
    done = torch.ones(B, dtype=torch.int64, device=dev)  # tokens of each sequence so far
    at = torch.arange(drafts + 1, device=dev)
    while int(done.min()) < steps:
        base, w = guess.lengths, guess.w
        tried, q, ws = [last], [], []
        for i in range(drafts + 1):  # the last of them only enters the draft model's cache
            p = probs(draft.extend(guess, tried[-1].clamp(min=0), keep=False)[:, 0])
            ws.append([x[..., 0] for x in guess._new])
            guess.keep(torch.ones_like(guess.lengths))
            if i < drafts:
                q.append(p)
                tried.append(_sample(p, uniform(B)))
        x = torch.cat(tried, 1)
        p = probs(model.extend(state, x.clamp(min=0), keep=False))
        n, next_tokens = verify_drafts(p, torch.stack(q, 1), x[:, 1:].contiguous(), uniform(B, drafts), uniform(B))
        kept = torch.where(done < steps, n + 1, 0)  # sequences that are done stay where they are
        state.keep(kept.to(torch.int32))
        guess.lengths, guess.w = base, w
        guess._new = [torch.stack(layer, 2) for layer in zip(*ws)]
        guess.keep(kept.to(torch.int32))
        places = torch.where(at < kept.unsqueeze(1), done.unsqueeze(1) + at, out.shape[1] - 1)
        out.scatter_(1, places, torch.where(at < kept.unsqueeze(1), next_tokens, out[:, -1:]))
        last = torch.where((kept > 0).unsqueeze(1), next_tokens.gather(1, n.unsqueeze(1)), last)
        done = done + kept
    return out[:, :steps]
