"""TextDecoderStack.prefill_packed where a prompt is not served: what it returns, and what it leaves as it was.

The restatement is the same decoder on slot caches, prompt by prompt; the bound is the decoder tests' own for 16-bit
activations, 2e-2 of the largest logit."""
import pytest
import torch

from whisperdrz_amd import KVPagePool
from whisperdrz_amd.decoder import TextDecoderStack
from whisperdrz_amd.kv_cache import KVSlotPool

pytestmark = pytest.mark.gpu

N_VOCAB, N_CTX, N_STATE, N_HEAD, N_LAYER, AUDIO = 300, 80, 128, 2, 2, 50
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def stack(cuda):
    torch.manual_seed(5)
    stack = TextDecoderStack(N_VOCAB, N_CTX, N_STATE, N_HEAD, N_LAYER).requires_grad_(False)
    stack.positional_embedding.mul_(50.0)  # as large as the tokens': a wrong position is seen
    return stack.to(cuda, BF16).eval()


def pool(cuda, n_pages=60, streams=6):
    return KVPagePool(N_LAYER, streams, n_pages, N_HEAD, 64, N_CTX, AUDIO, BF16, cuda)


def prompts(cuda, lens, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return (torch.randint(0, N_VOCAB, (sum(lens),), generator=g, device=cuda), torch.tensor(lens, device=cuda),
            torch.randn(len(lens), AUDIO, N_STATE, generator=g, device=cuda).to(BF16))


def alone(cuda, stack, tokens, xa):
    """The logits of one prompt by itself."""
    slots = KVSlotPool(N_LAYER, 1, N_HEAD, 64, self_len=N_CTX, cross_len=AUDIO, dtype=BF16, device=cuda)
    return stack.prefill_flash(tokens[None], xa[None], slots.self_kv, slots.cross_kv, torch.zeros(1, dtype=torch.long, device=cuda))[0]


def close(a, b):
    a, b = a.float(), b.float()
    return bool(torch.isfinite(a).all()) and (a - b).abs().max().item() <= 2e-2 * max(b.abs().max().item(), 1.0)


@pytest.mark.parametrize("lens,named,n_pages,served", [
    ([16, 33, 17, 5], [0, 1, 2, 3], 4, [0, 0, -1, -1]),  # pages run out
    ([20, 9, 30, 40], [3, 3, -1, 6], 60, [0, -1, -1, -1]),  # named twice, no stream
    ([70, 81, 100, 3], [0, 1, 2, 4], 60, [0, -1, -1, 0])])  # longer than the decoder
def test_logits_of_prompts_that_are_not_served(cuda, stack, lens, named, n_pages, served):
    """A prompt without a cache has the logits that it has by itself; positions that the decoder does not have are NaN."""
    pages = pool(cuda, n_pages)
    tokens, new, xa = prompts(cuda, lens)
    logits, plan = stack.prefill_packed(tokens, new, xa, pages, torch.tensor(named, device=cuda))
    assert plan.starts.tolist() == served
    for i, (got, t) in enumerate(zip(logits.split(lens), tokens.split(lens))):
        assert close(got[:N_CTX], alone(cuda, stack, t[:N_CTX], xa[i])), i
        assert got[N_CTX:].isnan().all()


def test_cross_caches_of_prompts_that_are_not_served(cuda, stack):
    """The windows of prompts without pages, and of a stream's second prompt, go to no slot."""
    pages = pool(cuda, 4)
    for c in pages.cross_kv:
        c.k_cache.fill_(3.0), c.v_cache.fill_(3.0)
    lens, named = [16, 33, 17, 2, 5], [4, 0, 2, 4, 0]
    tokens, new, xa = prompts(cuda, lens, 1)
    logits, plan = stack.prefill_packed(tokens, new, xa, pages, torch.tensor(named, device=cuda))
    assert plan.starts.tolist() == [0, 0, -1, -1, -1]
    for block, c in zip(stack.blocks, pages.cross_kv):
        kv = torch.nn.functional.linear(xa, *block.cross_attn.kv_weight()).view(len(lens), AUDIO, 2, N_HEAD, 64)
        for s in range(6):
            want = kv[named.index(s)] if s in (0, 4) else torch.full_like(kv[0], 3.0)
            assert torch.equal(c.k_cache[s], want[:, 0]) and torch.equal(c.v_cache[s], want[:, 1]), s


def state(pages):
    t = pages.tables
    caches = [x for c in pages.self_kv for x in (c.k_pages, c.v_pages)] + [x for c in pages.cross_kv for x in (c.k_cache, c.v_cache)]
    return [x.clone() for x in (t.tables, t.page_counts, t.seq_lens, t.free_pages, t.n_free, *caches)]


def test_calls_that_are_refused_change_nothing(cuda, stack):
    """Windows that are not the cross caches' length (steps attend all of a slot's rows), and inputs of other types, devices and
    shapes: refused before a stream is emptied or a page is taken."""
    pages = pool(cuda)
    tokens, new, xa = prompts(cuda, [20, 9], 2)
    at = torch.tensor([1, 4], device=cuda)
    stack.prefill_packed(tokens, new, xa, pages, at)
    other = TextDecoderStack(N_VOCAB, N_CTX, N_STATE, N_HEAD, N_LAYER + 1).to(cuda, BF16)
    wide = TextDecoderStack(N_VOCAB, N_CTX, 2 * N_STATE, 2 * N_HEAD, N_LAYER).to(cuda, BF16)
    before = state(pages)
    for s, args, err in ((stack, (tokens, new, xa[:, :-1], pages, at), ValueError), (stack, (tokens, new, torch.cat([xa, xa], 1), pages, at), ValueError),
                         (stack, (tokens, new, xa.float(), pages, at), TypeError), (stack, (tokens, new, xa[..., :64], pages, at), ValueError),
                         (stack, (tokens, new, xa.cpu(), pages, at), RuntimeError), (stack, (tokens, new.cpu(), xa, pages, at), RuntimeError),
                         (stack, (tokens, new.float(), xa, pages, at), TypeError), (stack, (tokens.float(), new, xa, pages, at), TypeError),
                         (stack, (tokens, new, xa, pages, at.float()), TypeError), (stack, (tokens.cpu(), new, xa, pages, at), RuntimeError),
                         (stack, (tokens, new, xa, KVPagePool(N_LAYER, 6, 60, N_HEAD, 64, N_CTX, AUDIO, torch.float16, cuda), at), TypeError),
                         (other, (tokens, new, xa, pages, at), ValueError),
                         (wide, (tokens, new, torch.cat([xa, xa], 2), pages, at), ValueError)):
        with pytest.raises(err):
            s.prefill_packed(*args)
        assert all(torch.equal(a, b) for a, b in zip(before, state(pages)))


@pytest.mark.parametrize("lens,told,served", [
    ([16, 9, 12], [16, 9, 14], [0, 0, -1]), ([16, 9, 12], [16, 9 + 2**31 - 40, 12], [0, -1, -1]), ([16, 9, 12], [16, 9, 3], [0, 0, 0]),
    ([16, 9, 12], [16, -1, 12], [0, -1, 0])])
def test_lengths_that_do_not_match_the_tokens(cuda, stack, lens, told, served):
    """A prompt whose tokens are not all there takes nothing, nor do those behind it; tokens of no prompt have NaN."""
    pages = pool(cuda)
    tokens, _, xa = prompts(cuda, lens, 3)
    at = torch.tensor([2, 5, 0], device=cuda)
    logits, plan = stack.prefill_packed(tokens, torch.tensor(told, device=cuda), xa, pages, at)
    assert plan.starts.tolist() == served
    held = [n if s == 0 else 0 for n, s in zip(told, served)]
    assert pages.tables.seq_lens[at].tolist() == held and 60 - int(pages.tables.n_free) == sum(-(-n // 16) for n in held)
    a = 0
    for i, n in enumerate(held):
        if n:
            assert close(logits[a : a + n], alone(cuda, stack, tokens[a : a + n], xa[i]))
        a += n
    assert logits[a:].isnan().all() and (plan.slots[a:] == -1).all()


def test_steps_that_are_refused_change_nothing(cuda, stack):
    """A step on caches that do not fit the decoder, or with streams that do not fit its rows, takes no place for its tokens."""
    pages = pool(cuda)
    tokens, new, xa = prompts(cuda, [20, 9], 4)
    at = torch.tensor([1, 4], device=cuda)
    stack.prefill_packed(tokens, new, xa, pages, at)
    before = state(pages)
    wide = TextDecoderStack(N_VOCAB, N_CTX, 2 * N_STATE, 2 * N_HEAD, N_LAYER).to(cuda, BF16)
    half = TextDecoderStack(N_VOCAB, N_CTX, N_STATE, N_HEAD, N_LAYER).to(cuda, torch.float16)
    two, pos = torch.zeros(2, 1, dtype=torch.long, device=cuda), torch.tensor([20, 9], device=cuda)
    elsewhere = pool(cuda)
    mixed = KVPagePool(N_LAYER, 6, 60, N_HEAD, 64, N_CTX, AUDIO, torch.float16, cuda)
    for s, args, err in ((stack, (two, pages.self_kv[:1], pages.cross_kv, pos, at), ValueError), (stack, (two, pages.self_kv, pages.cross_kv[:1], pos, at), ValueError),
                         (stack, (two, [pages.self_kv[0], elsewhere.self_kv[1]], pages.cross_kv, pos, at), ValueError),
                         (stack, (two, pages.self_kv, mixed.cross_kv, pos, at), TypeError), (wide, (two, pages.self_kv, pages.cross_kv, pos, at), ValueError),
                         (half, (two, pages.self_kv, pages.cross_kv, pos, at), TypeError), (stack, (two, pages.self_kv, pages.cross_kv, pos, at[:1]), ValueError),
                         (stack, (two, pages.self_kv, pages.cross_kv, pos, torch.tensor([1, 4, 0], device=cuda)), ValueError)):
        with pytest.raises(err):
            s.forward_flash(*args)
        assert all(torch.equal(a, b) for a, b in zip(before, state(pages)))


@pytest.mark.parametrize("lens,n", [([0, 5, 0], 5), ([0, 0], 0), ([], 0), ([], 3)])
def test_prompts_without_tokens(cuda, stack, lens, n):
    """Their windows are kept, so that a first step gives what it gives after a prompt into slots; without streams nothing is."""
    pages = pool(cuda)
    tokens, new, xa = prompts(cuda, lens or [n], 6)
    if not lens:
        new, xa = new[:0], xa[:0]
    at = torch.tensor([5, 2, 3][: len(lens)], dtype=torch.long, device=cuda)
    logits, plan = stack.prefill_packed(tokens, new, xa, pages, at)
    assert logits.shape == (n, N_VOCAB) and plan.starts.tolist() == [0] * len(lens)
    assert bool(logits.isfinite().all()) if lens else bool(logits.isnan().all())
    step = torch.randint(0, N_VOCAB, (len(lens), 1), device=cuda)
    got = stack.forward_flash(step, pages.self_kv, pages.cross_kv, new, at)
    assert got.shape == (len(lens), 1, N_VOCAB)
    a = 0
    for i, m in enumerate(lens):
        assert close(got[i], alone(cuda, stack, torch.cat([tokens[a : a + m], step[i]]), xa[i])[-1:])
        a += m


def test_tokens_of_32_bits_and_other_tables(cuda, stack):
    """Tokens and a decoder that the fused first operation does not take have the same logits."""
    lens, named, told = [16, 33, 17, 5], [0, 1, 1, 6], [16, 33, 17, 3]
    tokens, new, xa = prompts(cuda, lens, 7)
    new = torch.tensor(told, device=cuda)
    at = torch.tensor(named, device=cuda)
    want, plan = stack.prefill_packed(tokens, new, xa, pool(cuda), at)
    got, other = stack.prefill_packed(tokens.int(), new.short(), xa, pool(cuda), at.int())
    assert torch.equal(got.isnan(), want.isnan()) and bool(want[:-2].isfinite().all()) and bool(want[-2:].isnan().all())
    assert close(got[:-2], want[:-2]) and all(torch.equal(a, b) for a, b in zip(plan, other))
