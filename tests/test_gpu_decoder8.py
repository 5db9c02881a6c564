"""The decoder with 8-bit caches (KVSlotPool(cache_bits=8)) and 4-bit Linears
(TextDecoderStack.quantize_linears_), as a program uses them: prompt, single steps, a verified draft that is
partly rejected, and captured steps.

The restatement runs the same modules on fp32 weights that the codes stand for and attends in fp32 torch over the
values that its own cache stands for (whose bits the cache's tests pin down), so both round the same
things; the bound is the decoder tests' own for 16-bit activations, 2e-2 of the largest logit.
"""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

N_VOCAB, N_CTX, N_STATE, N_HEAD, N_LAYER, CROSS_LEN = 512, 80, 256, 4, 2, 50


class _Dequantized(nn.Module):
    def __init__(self, q):
        super().__init__()
        self.w, self.b = q.dequantize(), None if q.bias is None else q.bias.float()
        self.in_features, self.out_features, self.bias = q.in_features, q.out_features, q.bias

    def forward(self, x):
        y = x.float() @ self.w.T
        return (y if self.b is None else y + self.b).to(x.dtype)


def _attend(cache, lens, at, q, k, v, scale):
    """fp32 attention over what ``cache`` stands for at ``lens`` (None: all of a cross cache), then the append."""
    keys, values = cache.dequantize(None if lens is None else torch.zeros_like(cache.seq_lens).index_copy_(0, at, lens))
    out = torch.empty_like(q)
    for b, slot in enumerate(at.tolist()):
        n = cache.max_seq_length if lens is None else int(lens[b])
        kk, vv = keys[slot, :n], values[slot, :n]
        if k is not None:
            kk, vv = torch.cat([kk, k[b].float()]), torch.cat([vv, v[b].float()])
        s = torch.einsum("thd,lhd->htl", q[b].float(), kk) * scale
        if k is not None:
            T = q.shape[1]
            s = s + torch.triu(torch.full((T, n + T), float("-inf"), device=q.device), diagonal=n + 1)
        out[b] = torch.einsum("htl,lhd->thd", torch.softmax(s, -1), vv).to(q.dtype)
    if k is not None:
        for b, slot in enumerate(at.tolist()):
            cache._write(k[b:b + 1], v[b:b + 1], at[b:b + 1], int(lens[b]))
    return out


def _make(cuda, dtype, seed, bits, group=None, logits=False):
    """The stack, and its restatement."""
    from whisperdrz_amd.decoder import TextDecoderStack
    from whisperdrz_amd.decode_ops import QuantLinear4

    stacks = []
    for _ in range(2):
        torch.manual_seed(seed)
        stacks.append(TextDecoderStack(N_VOCAB, N_CTX, N_STATE, N_HEAD, N_LAYER).to(cuda, dtype).eval())
    hip, ref = stacks
    if group:
        hip.quantize_linears_(group, logits)
        ref.quantize_linears_(group, logits)
        for m in list(ref.modules()):
            for name, child in list(m.named_children()):
                if isinstance(child, QuantLinear4) and name not in ("qkv4", "logits4"):
                    setattr(m, name, _Dequantized(child))
        for blk in ref.blocks:
            for i in (0, 2):
                if isinstance(blk.mlp[i], QuantLinear4):
                    blk.mlp[i] = _Dequantized(blk.mlp[i])
        if logits:
            w = ref.logits4.dequantize()
            ref._logits = lambda h: (h.float() @ w.T).to(h.dtype)
    ref.fused_small_ops = False
    if bits == 8:
        for blk in ref.blocks:
            for m in (blk.attn, blk.cross_attn):
                m.cached = lambda q, c, k, v, lens, idx: _attend(c, lens, idx.long(), q, k, v, q.shape[-1] ** -0.5)
    return hip, ref


def _pool(cuda, dtype, n_slots, bits):
    from whisperdrz_amd.kv_cache import KVSlotPool

    return KVSlotPool(N_LAYER, n_slots, N_HEAD, 64, self_len=N_CTX, cross_len=CROSS_LEN, dtype=dtype, device=cuda,
                      cache_bits=bits)


def _close(a, b, what):
    a, b = a.float(), b.float()
    assert torch.isfinite(a).all(), what
    err, tol = (a - b).abs().max().item(), 2e-2 * max(b.abs().max().item(), 1.0)
    assert err <= tol, f"{what}: max|diff|={err:.3e} > {tol:.3e}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits,group,logits", [(8, None, False), (16, 64, False), (8, 32, True)])
def test_prompt_steps_and_drafts(cuda, dtype, bits, group, logits):
    hip, ref = _make(cuda, dtype, 3, bits, group, logits)
    B, slots = 3, torch.tensor([4, 0, 2], device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    xa = torch.randn(B, CROSS_LEN, N_STATE, generator=g, device=cuda).to(dtype)
    toks = lambda n: torch.randint(0, N_VOCAB, (B, n), generator=g, device=cuda)
    ph, pr = _pool(cuda, dtype, 5, bits), _pool(cuda, dtype, 5, bits)
    with torch.no_grad():
        prompt = toks(29)
        _close(hip.prefill_flash(prompt, xa, ph.self_kv, ph.cross_kv, slots),
               ref.prefill_flash(prompt, xa, pr.self_kv, pr.cross_kv, slots), "prompt")
        for n, accepted in ((1, 1), (1, 1), (5, 2), (1, 1), (5, 5), (1, 1)):
            t = toks(n)
            pos = ph.self_kv[0].seq_lens[slots].long()[:, None] + torch.arange(n, device=cuda)
            _close(hip.forward_flash(t, ph.self_kv, ph.cross_kv, pos, slots),
                   ref.forward_flash(t, pr.self_kv, pr.cross_kv, pos, slots), f"{n} tokens")
            for pool in (ph, pr):
                pool.self_seq_lens[:, slots] -= n - accepted
        assert torch.equal(ph.self_seq_lens, pr.self_seq_lens)


@pytest.mark.parametrize("rows", [1, 3, 6])
def test_captured_steps(cuda, rows):
    from whisperdrz_amd.decoder import BucketedDecodeGraphs

    dtype = torch.bfloat16
    hip, _ = _make(cuda, dtype, 7, 8, 64, True)
    pools = [_pool(cuda, dtype, 9, 8) for _ in range(2)]
    g = torch.Generator(device=cuda).manual_seed(2)
    xa = torch.randn(rows, CROSS_LEN, N_STATE, generator=g, device=cuda).to(dtype)
    slots = torch.randperm(8, generator=g, device=cuda)[:rows]
    with torch.no_grad():
        graphs = BucketedDecodeGraphs(hip, pools[0], N_VOCAB, buckets=[4, 8])
        for b in (4, 8):
            graphs.capture(b)
            graphs.static[b]["slots"].fill_(8)  # the padding's slot
        pools[0].reset()
        prompt = torch.randint(0, N_VOCAB, (rows, 28), generator=g, device=cuda)
        for p in pools:
            hip.prefill_flash(prompt, xa, p.self_kv, p.cross_kv, slots)
        for step in range(8):
            t = torch.randint(0, N_VOCAB, (rows, 1), generator=g, device=cuda)
            pos = pools[0].self_kv[0].seq_lens[slots].long()
            got = graphs.forward(t, pos, slots).clone()
            want = hip.forward_flash(t, pools[1].self_kv, pools[1].cross_kv, pos, slots)
            torch.cuda.synchronize()
            # another batch is another split of the sums; the caches' bits follow the activations'
            _close(got, want, f"step {step}")
            pools[0].self_seq_lens[:, 8] = 0
        assert torch.equal(pools[0].self_seq_lens[:, :8], pools[1].self_seq_lens[:, :8])


def test_quantized_layers_share_the_fused_projection(cuda):
    hip, _ = _make(cuda, torch.bfloat16, 1, 16, 64)
    a = hip.blocks[0].attn
    x = torch.randn(5, N_STATE, device=cuda).to(torch.bfloat16)
    from whisperdrz_amd import linear4

    whole = linear4(x, a.qkv4).view(5, 3, N_STATE)
    for i, m in enumerate((a.query, a.key, a.value)):
        assert torch.equal(linear4(x, m), whole[:, i]) and m.packed.data_ptr() == a.qkv4.packed[i * N_STATE // 16].data_ptr()
    # the uncached path runs on the same layers
    toks = torch.randint(0, N_VOCAB, (2, 9), device=cuda)
    xa = torch.randn(2, CROSS_LEN, N_STATE, device=cuda).to(torch.bfloat16)
    with torch.no_grad():
        assert torch.isfinite(hip(toks, xa)).all()


def test_quantize_refusals(cuda):
    from whisperdrz_amd.decoder import TextDecoderStack

    hip, _ = _make(cuda, torch.bfloat16, 1, 16, 64)
    with pytest.raises(ValueError, match="already"):
        hip.quantize_linears_(64)
    odd = TextDecoderStack(64, 16, 192, 3, 1).to(cuda, torch.bfloat16)
    with pytest.raises(NotImplementedError, match="group"):
        odd.quantize_linears_(128)
    assert isinstance(odd.blocks[0].attn.query, nn.Linear)  # nothing was changed
    with pytest.raises(TypeError):
        TextDecoderStack(64, 16, 192, 3, 1).quantize_linears_(64)
