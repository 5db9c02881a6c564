"""The decoder on paged self caches, as a program uses them: packed prompts of different lengths, scored tokens, single
steps, a draft that is partly rejected, captured steps, streams that end and others that take their pages.

The restatement is the same decoder on slot caches, prompt by prompt; the bound is the decoder tests' own for 16-bit
activations, 2e-2 of the largest logit."""
import pytest
import torch

from oracle.paged_oracle import logprobs

pytestmark = pytest.mark.gpu

N_VOCAB, N_CTX, N_HEAD, N_LAYER, CROSS_LEN = 512, 80, 4, 2, 50


def _make(cuda, dtype, group=None, n_state=256):
    from whisperdrz_amd.decoder import TextDecoderStack

    torch.manual_seed(3)
    stack = TextDecoderStack(N_VOCAB, N_CTX, n_state, N_HEAD, N_LAYER).to(cuda, dtype).eval()
    return stack.quantize_linears_(group) if group else stack


def _pools(cuda, dtype, n_pages=40, n_state=256, streams=6):
    from whisperdrz_amd import KVPagePool
    from whisperdrz_amd.kv_cache import KVSlotPool

    d = n_state // N_HEAD
    return (KVPagePool(N_LAYER, streams, n_pages, N_HEAD, d, N_CTX, CROSS_LEN, dtype, cuda),
            KVSlotPool(N_LAYER, streams, N_HEAD, d, self_len=N_CTX, cross_len=CROSS_LEN, dtype=dtype, device=cuda))


def _close(a, b, what):
    a, b = a.float(), b.float()
    assert torch.isfinite(a).all(), what
    err, tol = (a - b).abs().max().item(), 2e-2 * max(b.abs().max().item(), 1.0)
    assert err <= tol, f"{what}: max|diff|={err:.3e} > {tol:.3e}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [None, 64])
def test_prompts_scores_steps_and_drafts(cuda, dtype, group):
    from whisperdrz_amd import token_logprobs

    stack = _make(cuda, dtype, group)
    pages, slots = _pools(cuda, dtype)
    at, lens = torch.tensor([4, 0, 2, 5], device=cuda), [17, 1, 40, 16]
    g = torch.Generator(device=cuda).manual_seed(1)
    xa = torch.randn(4, CROSS_LEN, 256, generator=g, device=cuda).to(dtype)
    tokens = torch.randint(0, N_VOCAB, (sum(lens),), generator=g, device=cuda)
    with torch.no_grad():
        got, plan = stack.prefill_packed(tokens, torch.tensor(lens, device=cuda), xa, pages, at)
        want = [stack.prefill_flash(t[None], xa[i : i + 1], slots.self_kv, slots.cross_kv, at[i : i + 1])[0]
                for i, t in enumerate(tokens.split(lens))]
        _close(got, torch.cat(want), "prompts")
        assert plan.starts.tolist() == [0] * 4 and pages.tables.seq_lens[at].tolist() == lens
        # what the prompt's logits say of the tokens that follow
        scores = token_logprobs(got, tokens, top=3)
        lp, entropy, values, ids = logprobs(got.cpu(), tokens.cpu(), 3)
        assert torch.equal(scores.top_ids.cpu(), ids)
        for a, b in ((scores.logprobs, lp), (scores.entropy, entropy), (scores.top_logprobs, values)):
            assert torch.allclose(a.cpu().double(), b, rtol=2**-17, atol=2.0**-92)
        for n, accepted in ((1, 1), (5, 2), (1, 1), (4, 4), (1, 1)):
            t = torch.randint(0, N_VOCAB, (4, n), generator=g, device=cuda)
            pos = slots.self_kv[0].seq_lens[at].long()[:, None] + torch.arange(n, device=cuda)
            assert torch.equal(pages.tables.seq_lens[at].long(), pos[:, 0])
            _close(stack.forward_flash(t, pages.self_kv, pages.cross_kv, pos, at),
                   stack.forward_flash(t, slots.self_kv, slots.cross_kv, pos, at), f"{n} tokens")
            slots.self_seq_lens[:, at] -= n - accepted
            pages.tables.truncate(pages.tables.seq_lens[at] - (n - accepted), at)
        free = int(pages.tables.n_free)
        held = sum(-(-n // 16) for n in pages.tables.seq_lens.tolist())
        assert free + held == 40
        pages.release(at[:2])
        assert pages.tables.seq_lens[at].tolist()[:2] == [0, 0]
        pages.release()
        assert int(pages.tables.n_free) == 40 and sorted(pages.tables.free_pages.tolist()) == list(range(40))


def test_one_row_and_streams_in_order(cuda):
    """A single stream (the small step's own path), and rows that are streams 0, 1, .. without a slot map."""
    stack = _make(cuda, torch.bfloat16)
    pages, slots = _pools(cuda, torch.bfloat16)
    g = torch.Generator(device=cuda).manual_seed(2)
    for B in (1, 6):
        xa = torch.randn(B, CROSS_LEN, 256, generator=g, device=cuda).bfloat16()
        prompt = torch.randint(0, N_VOCAB, (B, 7), generator=g, device=cuda)
        at = torch.arange(B, device=cuda)
        with torch.no_grad():
            got, _ = stack.prefill_packed(prompt.view(-1), torch.full((B,), 7, device=cuda), xa, pages, at)
            want = stack.prefill_flash(prompt, xa, slots.self_kv, slots.cross_kv, at)
            _close(got.view_as(want), want, "prompt")
            for i in range(12):
                t = torch.randint(0, N_VOCAB, (B, 1), generator=g, device=cuda)
                pos = torch.full((B,), 7 + i, device=cuda)
                _close(stack.forward_flash(t, pages.self_kv, pages.cross_kv, pos), stack.forward_flash(t, slots.self_kv, slots.cross_kv, pos), "step")


def test_captured_steps_change_only_their_streams(cuda):
    from whisperdrz_amd.decoder import BucketedDecodeGraphs

    stack = _make(cuda, torch.bfloat16)
    pages, slots = _pools(cuda, torch.bfloat16)
    at, lens = torch.tensor([5, 1, 3], device=cuda), [15, 30, 2]
    g = torch.Generator(device=cuda).manual_seed(3)
    xa = torch.randn(3, CROSS_LEN, 256, generator=g, device=cuda).bfloat16()
    tokens = torch.randint(0, N_VOCAB, (sum(lens),), generator=g, device=cuda)
    with torch.no_grad():
        stack.prefill_packed(tokens, torch.tensor(lens, device=cuda), xa, pages, at)
        for i, t in enumerate(tokens.split(lens)):
            stack.prefill_flash(t[None], xa[i : i + 1], slots.self_kv, slots.cross_kv, at[i : i + 1])
        state = [x.clone() for x in (pages.tables.tables, pages.tables.seq_lens, pages.tables.free_pages, pages.self_kv[1].k_pages)]
        graphs = BucketedDecodeGraphs(stack, pages, N_VOCAB, buckets=[2, 4])
        graphs.capture(4)
        graphs.capture(2)
        now = (pages.tables.tables, pages.tables.seq_lens, pages.tables.free_pages, pages.self_kv[1].k_pages)
        assert all(torch.equal(a, b) for a, b in zip(state, now))
        pos = torch.tensor(lens, device=cuda)
        for i in range(20):  # page borders of every stream pass by
            rows = torch.arange(3, device=cuda) if i % 3 else torch.tensor([2, 0], device=cuda)
            t = torch.randint(0, N_VOCAB, (len(rows), 1), generator=g, device=cuda)
            got = graphs.forward(t, pos[rows], at[rows])
            _close(got, stack.forward_flash(t, slots.self_kv, slots.cross_kv, pos[rows], at[rows]), f"step {i}")
            pos[rows] += 1
            assert torch.equal(pages.tables.seq_lens[at], pos.int()) and pages.tables.seq_lens.sum() == pos.sum()
        assert graphs.hits[4] > 0 and graphs.hits[2] > 0 and graphs.misses == 0


def test_pages_run_out(cuda):
    """A prompt without pages has no cache, the others are served; a step without a page is NaN for its row alone."""
    stack = _make(cuda, torch.float16)
    pages, _ = _pools(cuda, torch.float16, n_pages=4)
    at = torch.tensor([0, 1, 2], device=cuda)
    xa = torch.randn(3, CROSS_LEN, 256, device=cuda).half()
    tokens = torch.randint(0, N_VOCAB, (16 + 33 + 16,), device=cuda)
    with torch.no_grad():
        logits, plan = stack.prefill_packed(tokens, torch.tensor([16, 33, 16], device=cuda), xa, pages, at)
        assert plan.starts.tolist() == [0, 0, -1] and logits.isfinite().all() and (plan.slots[-16:] == -1).all()
        assert pages.tables.seq_lens.tolist()[:3] == [16, 33, 0] and int(pages.tables.n_free) == 0
        step = stack.forward_flash(torch.zeros(2, 1, dtype=torch.long, device=cuda), pages.self_kv, pages.cross_kv,
                                   torch.tensor([16, 33], device=cuda), at[:2])
        assert step[0].isnan().all() and step[1].isfinite().all() and pages.tables.seq_lens.tolist()[:2] == [16, 34]
        pages.release(at[1:2])
        step = stack.forward_flash(torch.zeros(1, 1, dtype=torch.long, device=cuda), pages.self_kv, pages.cross_kv,
                                   torch.tensor([16], device=cuda), at[:1])
        assert step.isfinite().all() and int(pages.tables.n_free) == 2


def test_refusals(cuda):
    stack = _make(cuda, torch.bfloat16)
    pages, _ = _pools(cuda, torch.bfloat16)
    xa, at = torch.zeros(2, CROSS_LEN, 256, device=cuda).bfloat16(), torch.tensor([0, 1], device=cuda)
    tokens, lens = torch.zeros(5, dtype=torch.long, device=cuda), torch.tensor([2, 3], device=cuda)
    for args in ((tokens[None], lens, xa, pages, at), (tokens, lens[:1], xa, pages, at), (tokens, lens, xa, pages, at[:1])):
        with pytest.raises(ValueError):
            stack.prefill_packed(*args)
    stack.fused_small_ops = False
    with pytest.raises(NotImplementedError):
        stack.prefill_packed(tokens, lens, xa, pages, at)
    with pytest.raises(NotImplementedError):
        stack.forward_flash(tokens[:2, None], pages.self_kv, pages.cross_kv, at, at)
