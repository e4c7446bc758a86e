"""The decoder answering: prompts into the caches, single tokens, drafts and samples behind one prompt, against the logits of
the whole sequence (the training path's)."""
import pytest
import torch

from fpa.lm import FPADecoder, generate

TINY = dict(vocab=97, d_model=64, n_heads=2, layers=2, d_mlp=128)


def model(dev, seed=0, **over):
    torch.manual_seed(seed)
    return FPADecoder(**{**TINY, **over}).to(dev).eval()


def devices():
    return ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def need(dev):
    if dev == "cuda" and not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    print(f"[generate] {dev}", flush=True)


# Two layers in fp32: the logits of order 1 here come from the same sums in another order, a few hundred terms each of relative
# rounding 2^-24 through two layers; 1e-3 leaves a factor of ten over (2 layers * 300 terms * 2^-24 * |values| of 10).
TOL = 1e-3


@pytest.mark.parametrize("dev", devices())
def test_steps_give_the_logits_of_the_whole_sequence(dev):
    """Ragged prompts, then 1, 3 and 17 tokens at a time, some rejected in between."""
    need(dev)
    m = model(dev)
    g = torch.Generator().manual_seed(1)
    B, T = 3, 90
    full = torch.randint(0, 97, (B, 140), generator=g).to(dev)
    counts = torch.tensor([90, 1, 64], dtype=torch.int32, device=dev)
    with torch.no_grad():
        want = m(full)
    rows = torch.arange(B, device=dev)

    def near(a, at):
        assert (a - want[rows, at]).abs().max() <= TOL
    logits, state = m.start(full[:, :T], room=60, counts=counts)
    near(logits, counts.long() - 1)
    for n, keep in ((1, 1), (3, 2), (17, 17), (2, 1), (1, 1)):
        at = state.lengths.long()
        new = torch.stack([full[b, at[b]:at[b] + n] for b in range(B)])
        if keep < n:
            new[:, keep:] = 5  # rejected drafts leave nothing behind
        out = m.extend(state, new, keep=False)
        state.keep(torch.full_like(state.lengths, keep))
        for i in range(keep):
            near(out[:, i], at + i)
    assert state.lengths.tolist() == [112, 23, 86]


@pytest.mark.parametrize("dev", devices())
def test_samples_share_their_prompt(dev):
    need(dev)
    m = model(dev)
    g = torch.Generator().manual_seed(2)
    prompt, more = torch.randint(0, 97, (1, 75), generator=g).to(dev), torch.randint(0, 97, (5, 9), generator=g).to(dev)
    logits, state = m.start(prompt, room=20, samples=5)
    with torch.no_grad():
        want = m(torch.cat((prompt.expand(5, -1), more), 1))
    assert (logits - want[:, 74]).abs().max() <= TOL
    got = torch.cat([m.extend(state, more[:, :1]), m.extend(state, more[:, 1:5]), m.extend(state, more[:, 5:])], 1)
    assert (got - want[:, 75:]).abs().max() <= TOL
    assert state.prefix[1] == 75 and state.caches[0].pages == 2 + 5


@pytest.mark.parametrize("dev", devices())
@pytest.mark.parametrize("store", [None, torch.float8_e4m3fn])
def test_generate(dev, store):
    """All ways to sample run and stay inside the vocabulary; the same generator gives the same tokens."""
    need(dev)
    m, d = model(dev), model(dev, 1, layers=1)
    tokens = torch.randint(0, 97, (3, 40), generator=torch.Generator().manual_seed(3)).to(dev)
    counts = torch.tensor([40, 7, 33], dtype=torch.int32, device=dev)

    def run(**kw):
        return generate(m, kw.pop("tokens", tokens), 23, generator=torch.Generator(dev).manual_seed(4), store=store, **kw)
    for kw in (dict(counts=counts), dict(tokens=tokens[:1], samples=4), dict(counts=counts, draft=d, drafts=3),
               dict(tokens=tokens[:1], samples=2, draft=d)):
        out = run(**kw)
        assert out.shape[1] == 23 and ((out >= 0) & (out < 97)).all()
        assert torch.equal(out, run(**kw))


@pytest.mark.parametrize("dev", devices())
def test_a_model_accepts_its_own_drafts(dev):
    """With the model as its own draft nearly every draft is accepted (their probabilities agree to rounding), so that a
    round gives drafts + 1 tokens: at most two more rounds than that."""
    need(dev)
    m = model(dev)
    tokens = torch.randint(0, 97, (2, 30), generator=torch.Generator().manual_seed(5)).to(dev)
    calls = []
    extend = m.extend
    m.extend = lambda state, x, keep=True: calls.append(x.shape[1]) or extend(state, x, keep)
    generate(m, tokens, 41, draft=m, drafts=4, generator=torch.Generator(dev).manual_seed(6))
    assert calls.count(5) <= 8 + 2


def test_generate_refuses():
    m = model("cpu")
    tokens = torch.zeros(2, 5, dtype=torch.int64)
    for kw in (dict(steps=0), dict(steps=3, temperature=0.0), dict(steps=3, draft=m, drafts=0), dict(steps=3, samples=2)):
        with pytest.raises(ValueError):
            generate(m, tokens, **kw)


@pytest.mark.gpu
def test_half_precision_decoding_at_the_layers_size():
    """One layer of the 12-head model under fp16 autocast: prompt of 300, then tokens one at a time, fp16 and 8-bit caches, against the
    dense layer in fp32.  fp16 products and activations: 2^-11 a rounding, a few in a row, of values of order 1; 8 bits: each
    row's values are off by at most 2^-4 of themselves, which averages over hundreds of keys."""
    need("cuda")
    m = FPADecoder(vocab=997, d_model=768, n_heads=12, layers=1, d_mlp=1024).cuda().eval()
    tokens = torch.randint(0, 997, (2, 310), generator=torch.Generator().manual_seed(7)).cuda()
    with torch.no_grad():
        want = m(tokens)
    for store, tol in ((None, 1e-2), (torch.float8_e4m3fn, 5e-2)):
        with torch.autocast("cuda", dtype=torch.float16):
            logits, state = m.start(tokens[:, :300], room=16, store=store)
            got = [logits.unsqueeze(1)] + [m.extend(state, tokens[:, i:i + 1]) for i in range(300, 310)]
        got = torch.cat(got, 1).float()
        assert ((got - want[:, 299:]).norm() / want[:, 299:].norm()).item() <= tol


def test_samples_are_of_one_whole_prompt():
    m = model("cpu")
    tokens = torch.zeros(1, 7, dtype=torch.int64)
    with pytest.raises(ValueError, match="whole prompt"):
        m.start(tokens, 4, counts=torch.tensor([3]), samples=2)
    with pytest.raises(ValueError, match="samples"):
        m.start(tokens, 4, samples=0)
    with pytest.raises(ValueError, match="prompt"):
        m.start(tokens[:, :0], 4)
    with pytest.raises(ValueError, match="room"):
        m.start(tokens, -1)
    logits, state = m.start(tokens, 0, samples=2)  # no room: a table of one page all the same
    assert logits.shape[0] == 2 and state.table.shape == (2, 1)


@pytest.mark.parametrize("count", [0, 8, -1])
def test_counts_outside_the_prompt_are_refused(count):
    m = model("cpu")
    with pytest.raises(ValueError, match="counts"):
        m.start(torch.zeros(2, 7, dtype=torch.int64), 4, counts=torch.tensor([3, count]))


def test_an_empty_prompt_of_a_layer_ends_at_zero():
    """W starts at zero before a sequence's first position: extending a prompt of no positions is beginning a sequence."""
    a = model("cpu").blocks[0].attn
    x = torch.randn(2, 5, 64, generator=torch.Generator().manual_seed(3))
    cache = a.new_cache(2, x)
    table, counts = torch.tensor([[0], [1]], dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32)
    _, w = a.prompt(x, cache, table, counts)
    assert torch.equal(w[0], torch.zeros_like(w[0]))
    y, _ = a.extend(x, cache, table, torch.zeros_like(counts), torch.zeros_like(w))
    with torch.no_grad():
        assert (y - a(x)).abs().max() <= TOL


@pytest.mark.parametrize("drafted", [False, True])
def test_logits_without_a_distribution_give_no_token(drafted):
    """-1 in the answer, as verify_drafts gives it; it is never looked up as a token."""
    m = model("cpu")
    with torch.no_grad():
        m.head.weight.fill_(float("nan"))
    out = generate(m, torch.zeros(2, 5, dtype=torch.int64), 4, draft=model("cpu", 1, layers=1) if drafted else None, drafts=2)
    assert torch.equal(out, torch.full((2, 4), -1))
    if drafted:  # and drafts without one are none: the model's own tokens
        out = generate(model("cpu"), torch.zeros(2, 5, dtype=torch.int64), 4, draft=m, drafts=2)
        assert (out >= 0).all()
