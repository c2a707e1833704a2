"""GPU: what the decoder layers do with the attention's output."""
import pytest
import torch

from test_gpu_attention import no_device_error

pytestmark = pytest.mark.gpu


def test_decoder_stack_forward_after_the_attention(cuda):
    """From every layer's attention output on, the operators one after another give the next layer's q|k|v, the residual
    stream and the greedy tokens that the step gave: the same bits, as they are the same kernels."""
    from helios_b200 import attention as A
    from helios_b200.quantized import quantized_matmul, quantized_matmul_geglu, rms_norm, rms_norm_residual, synth_normal
    from helios_b200.stack import DecoderStack, StackConfig, decode_keys
    d, layers = 64, 5
    cfg = StackConfig(layers=layers, hidden=512, q_out=4 * d, kv_out=2 * d, inter=1024, vocab=2048)
    st = DecoderStack(cfg)
    st.attach_attention(40, 16, head_dim=d, window=40)
    scalars = [float(L["scalar"]) for L in st.layers]
    assert len(set(scalars)) > 2
    weights = [L[k] for L in st.layers for k in ("in_norm", "post_attn", "pre_ffn", "post_ffn")] + [st.final_norm]
    assert all(not torch.equal(a, b) for i, a in enumerate(weights) for b in weights[:i])
    table = torch.arange(36, dtype=torch.int32, device="cuda").reshape(3, 12)
    have = [0, 0, 0]
    for q_lens in ([70, 9, 3], [1, 1, 1], [5, 5, 5], [1, 150, 1]):
        have = [a + b for a, b in zip(have, q_lens)]
        off = [sum(q_lens[:b]) for b in range(4)]
        batch = A.PagedBatch(torch.tensor(off, dtype=torch.int32, device="cuda"),
                             torch.tensor(have, dtype=torch.int32, device="cuda"), table, max_q=max(q_lens))
        M = off[-1]
        h = synth_normal(200 + M, (M, cfg.hidden))
        rows = torch.tensor([o - 1 for o in off[1:]] * 7, device="cuda")          # more than one call of the LM head takes
        keep = []
        keys, res = st.forward(h, batch, rows=rows, keep=keep)
        no_device_error()
        x = h
        for L, kept, scalar in zip(st.layers, keep, scalars):
            assert torch.equal(kept["qkv"], quantized_matmul(rms_norm(x, L["in_norm"], cfg.eps), L["qkv"]))
            a = rms_norm_residual(quantized_matmul(kept["attn"].flatten(1), L["o"]), L["post_attn"], x, eps=cfg.eps)
            y = torch.empty((M, L["gu"].rows), dtype=torch.bfloat16, device="cuda") if M <= 16 else None
            down = quantized_matmul(quantized_matmul_geglu(rms_norm(a, L["pre_ffn"], cfg.eps), L["gu"], y=y), L["down"])
            before = x
            x = rms_norm_residual(down, L["post_ffn"], a, L["scalar"], cfg.eps)
            # the residual tails themselves, by their formula: norm, weight, sum and scalar round to bf16 once each, a
            # half step (2^-8 at most) of the value that they round, none of which is larger than the terms' sum
            for got, t, w, r, f in ((a, quantized_matmul(kept["attn"].flatten(1), L["o"]), L["post_attn"], before, 1.0),
                                    (x, down, L["post_ffn"], a, scalar)):
                t, w, r = t.double(), w.double(), r.double()
                n = t / torch.sqrt((t * t).mean(-1, keepdim=True) + cfg.eps) * w
                size = (n.abs() + r.abs()) * f
                assert ((got.double() - (r + n) * f).abs() <= 4 * 2.0 ** -8 * 1.02 * size + 2.0 ** -126).all()
        assert torch.equal(res, x)
        last = rms_norm(x[rows], st.final_norm, cfg.eps)
        logits = cfg.softcap * torch.tanh(quantized_matmul(last, st.lm).double() / cfg.softcap)
        tokens, _ = decode_keys(keys)
        mine = logits[torch.arange(len(rows)), torch.tensor(tokens)]
        # the greedy one, up to a rounding of either logit before the soft cap and after it, 2^-8 each
        top = logits.amax(-1)
        assert (top - mine <= 4 * 2.0 ** -8 * top.abs()).all()
        assert len(set(tokens)) > 1
    st.free()


def test_decoder_stack_forward_without_rows_or_tokens(cuda):
    """A step that wants no token (a chunk in the middle of a prompt), and one without new tokens."""
    from helios_b200 import attention as A
    from helios_b200.quantized import synth_normal
    from helios_b200.stack import DecoderStack, StackConfig
    st = DecoderStack(StackConfig(layers=2, hidden=512, q_out=256, kv_out=128, inter=1024, vocab=2048))
    st.attach_attention(8, 16, head_dim=64, window=0)
    int32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    h = synth_normal(7, (40, 512))
    batch = A.PagedBatch(int32([0, 40]), int32([40]), int32([[3, 1, 2]]), max_q=40)
    keys, res = st.forward(h, batch, rows=torch.empty(0, dtype=torch.int64, device="cuda"))
    none, again = st.forward(h, batch)
    assert keys.shape == (0,) and keys.dtype is torch.int64 and none is None and torch.equal(res, again)
    before = [L["cache"].k.clone() for L in st.layers]
    batch.q_offsets = int32([0, 0])
    keys, res = st.forward(h[:0], batch, rows=torch.empty(0, dtype=torch.int64, device="cuda"))
    assert keys.shape == (0,) and res.shape == (0, 512)
    assert all(torch.equal(a, L["cache"].k) for a, L in zip(before, st.layers))
    no_device_error()
    st.free()
