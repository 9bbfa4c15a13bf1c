"""The feed-forward half's operators as a block and a model run them, on a B200."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

OPTIONS = dict(ffn_impl="fused", ffn_activation="gelu", post_norm=True, residual_scale=0.5, residual_gate=True,
               counter_dropout=True)


def block(d=256, **kw):
    from dsalt.modules.dsalt_transformer import DSALTTransformerBlock
    torch.manual_seed(0)
    b = DSALTTransformerBlock(d_model=d, n_heads=4, n_min=8, n_max=64, k_lmk=8, max_seq_len=512, d_ff=520, layer_idx=3,
                              **kw).cuda()
    with torch.no_grad():
        for n, p in b.named_parameters():
            if n.endswith(("norm.weight", "post_weight")):
                p.normal_(1.0, 0.3)
    return b


def test_block_is_the_chain_of_its_operators():
    """A training block with every option gives, bit for bit, what its operators give when
    they are called one after another by hand; its gradients reach every parameter."""
    from dsalt import gated_ffn, residual_norm
    blk = block(dropout=0.25, **OPTIONS).train()
    cu = torch.tensor([0, 150, 333], dtype=torch.int32, device="cuda")
    seed = torch.tensor([77], dtype=torch.int64, device="cuda")
    x0 = torch.randn(333, 256, device="cuda").bfloat16()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        x = x0.clone().requires_grad_(True)
        y, _ = blk(x, cu_seqlens=cu, max_seqlen=183, cu_list=[0, 150, 333], dropout_seed=seed)
        h = blk.attn_norm(x0)
        a, _ = blk.attn(h, cu_seqlens=cu, max_seqlen=183, cu_list=[0, 150, 333])
        s = blk.attn_step
        x1, h2 = residual_norm(x0, a.to(x0.dtype), blk.ffn_norm.weight, post_weight=s.post_weight, scale=s.scale,
                               gate=torch.sigmoid(s.gate(h)))
        f = gated_ffn(h2, blk.ffn.gate_proj.weight, blk.ffn.up_proj.weight, blk.ffn.down_proj.weight, "gelu")
        s = blk.ffn_step
        ref, _ = residual_norm(x1, f, post_weight=s.post_weight, scale=s.scale, gate=torch.sigmoid(s.gate(h2)),
                               dropout_p=0.25, seed=seed, site=4)
    assert torch.equal(y, ref)
    y.float().square().mean().backward()
    for n, p in blk.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), n
    assert torch.isfinite(x.grad).all()


def test_operator_chain_against_64_bits():
    """residual_norm → gated_ffn → residual_norm: each operator's output, formed from the
    outputs that the operators before it gave, within its own rounding of the formula."""
    import torch.nn.functional as F
    from dsalt import gated_ffn, residual_norm
    T, d, f_ = 217, 320, 888
    g = torch.Generator(device="cuda").manual_seed(2)

    def n(*s, std=1.0, mean=0.0):
        return (torch.randn(*s, generator=g, device="cuda") * std + mean).bfloat16()

    x, a, w1, w2, sc = n(T, d), n(T, d), n(d, std=0.2, mean=1), n(d, std=0.2, mean=1), n(d, std=0.2, mean=0.5)
    wg, wu, wd = n(f_, d, std=d ** -0.5), n(f_, d, std=d ** -0.5), n(d, f_, std=f_ ** -0.5)
    x1, h = residual_norm(x, a, w1, scale=sc)
    f = gated_ffn(h, wg, wu, wd)
    x2, h2 = residual_norm(x1, f, w2, post_weight=w1)
    e = 2.0 ** -9 * (1 + 2.0 ** -7)  # a bf16 rounding, and the fp32 sums before it

    def norm(t, w):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w

    D = lambda t: t.double()  # noqa: E731
    s1, s2 = D(x) + D(sc) * D(a), D(x1) + norm(D(f), D(w1))
    for got, ref in ((x1, s1), (h, norm(s1, D(w1))), (x2, s2), (h2, norm(s2, D(w2)))):
        assert ((D(got) - ref).abs() <= 2 * e * ref.abs() + 2.0 ** -16).all()
    hid = F.silu(D(h) @ D(wg).t()) * (D(h) @ D(wu).t())
    ref = hid @ D(wd).t()
    # the hidden rows are rounded once (2^-8 of each), the sums carry 888·2^-22 of their terms
    bound = (2.0 ** -8 + f_ * 2.0 ** -22 + d * 2.0 ** -21) * (hid.abs() @ D(wd).abs().t()) + 2 * e * ref.abs() + 1e-3
    assert ((D(f) - ref).abs() <= bound).all()


@pytest.mark.parametrize("ckpt", [False, True])
def test_model_trains_with_the_operators(ckpt):
    """Finite loss, gradients for every parameter, the same step again from the same seed,
    another mask from another seed; evaluation drops nothing."""
    from dsalt.model import DSALTConfig, DSALTLMHeadModel
    torch.manual_seed(0)
    cfg = DSALTConfig(vocab_size=512, d_model=256, n_layers=2, n_heads=4, n_min=16, n_max=96, k_lmk=16, max_seq_len=512,
                      dropout=0.2, **OPTIONS)
    model = DSALTLMHeadModel.from_config(cfg).cuda().train()
    ids = torch.randint(0, 512, (600,), device="cuda")
    cu = torch.tensor([0, 300, 600], dtype=torch.int32, device="cuda")

    def step(seed):
        model.zero_grad(set_to_none=True)
        torch.manual_seed(seed)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = model(ids, cu_seqlens=cu, labels=ids, gradient_checkpointing=ckpt)["loss"]
        loss.backward()
        return loss.detach(), {k: p.grad.clone() for k, p in model.named_parameters()}

    la, ga = step(1)
    lb, gb = step(1)
    lc, _ = step(2)
    assert torch.isfinite(la) and torch.equal(la, lb) and not torch.equal(la, lc)
    for k, g in ga.items():
        assert torch.isfinite(g).all() and g.any(), k
    for k in ("layers.0.ffn_step.scale", "layers.1.ffn.gate_proj.weight"):  # no atomics on the way to these
        assert torch.equal(ga[k], gb[k]), k
    model.eval()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        a, b = (model(ids, cu_seqlens=cu)["logits"] for _ in range(2))
    assert torch.equal(a, b)


def test_fp32_model_with_steps_matches_plain_steps():
    """In fp32 (torch's feed-forward ops) a block with a post norm and a scale equals the
    same formula in torch's ops: fp32 rounding apart (2^-24 of each of some 40 operations on
    values of the residual stream's size)."""
    import torch.nn.functional as F
    blk = block(post_norm=True, residual_scale=0.3).eval()
    x = torch.randn(128, 256, device="cuda")
    cu = torch.tensor([0, 128], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        y, _ = blk(x, cu_seqlens=cu, max_seqlen=128, cu_list=[0, 128])

        def norm(t, w):
            return F.rms_norm(t, (256,), w, 1e-6)

        a, _ = blk.attn(norm(x, blk.attn_norm.weight), cu_seqlens=cu, max_seqlen=128, cu_list=[0, 128])
        x1 = x + blk.attn_step.scale * norm(a, blk.attn_step.post_weight)
        f = blk.ffn(norm(x1, blk.ffn_norm.weight))
        ref = x1 + blk.ffn_step.scale * norm(f, blk.ffn_step.post_weight)
    torch.testing.assert_close(y, ref, rtol=1e-4, atol=1e-4)


def test_fused_and_gemm_feed_forward_agree():
    """The two implementations differ by bf16 roundings: silu's, the hidden value's and the
    result's (gemm rounds gate, up and silu too): 6·2^-8 of the terms' magnitudes at most."""
    from dsalt.modules.dsalt_transformer import SwiGLUFFN
    torch.manual_seed(0)
    a, b = SwiGLUFFN(256, 704).cuda(), SwiGLUFFN(256, 704, impl="fused").cuda()
    b.load_state_dict(a.state_dict())
    x = torch.randn(3, 100, 256, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        ya, yb = a(x), b(x)
    assert ya.dtype == yb.dtype == torch.bfloat16 and ya.shape == yb.shape
    D = lambda t: t.detach().bfloat16().double()  # noqa: E731
    hid = torch.nn.functional.silu(D(x) @ D(a.gate_proj.weight).t()) * (D(x) @ D(a.up_proj.weight).t())
    mag = hid.abs() @ D(a.down_proj.weight).abs().t()
    assert ((ya.double() - yb.double()).abs() <= 6 * 2.0 ** -8 * mag + 1e-6).all()


def test_first_backward_of_a_process_may_be_a_gated_ffn():
    """A thread that has made no CUDA call yet can run the backward's tensor maps."""
    import threading
    from dsalt.kernels.gated_ffn import gated_ffn
    ts = [torch.randn(*s, device="cuda").bfloat16().requires_grad_(True) for s in ((70, 64), (96, 64), (96, 64), (64, 96))]
    got = []

    def work():
        y = gated_ffn(*ts)
        got.append(torch.autograd.grad(y, ts, torch.ones_like(y)))

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert len(got) == 1 and all(torch.isfinite(g).all() for g in got[0])


def test_first_call_of_a_process_inside_a_capture():
    """A captured call finds no status word yet: it makes none that would live in the graph."""
    from dsalt import gated_ffn
    from dsalt.kernels import dsalt_cuda
    ts = [torch.randn(*s, device="cuda").bfloat16() for s in ((400, 64), (96, 64), (96, 64), (64, 96))]
    ref = gated_ffn(*ts)
    saved = dict(dsalt_cuda._STATUS)
    dsalt_cuda._STATUS.clear()
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = gated_ffn(*ts)
        assert not dsalt_cuda._STATUS
    finally:
        dsalt_cuda._STATUS.update(saved)
    graph.replay()
    assert torch.equal(y, ref)
    dsalt_cuda.check_device_status(ref.device)


def test_offsets_past_32_bits():
    """More than 2^32 elements: the last rows equal the same rows of a small call (rows do not
    depend on one another; the feed-forward sums have one order in both tilings)."""
    from dsalt import gated_ffn, residual_norm
    d, T, n = 1024, (1 << 22) + 5, 700
    x, f = (torch.zeros(T, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    x[-n:], f[-n:] = torch.randn(n, d, device="cuda"), torch.randn(n, d, device="cuda")
    w = torch.rand(d, device="cuda") + 0.5
    big, small = residual_norm(x, f, w, post_weight=w), residual_norm(x[-n:], f[-n:], w, post_weight=w)
    assert all(torch.equal(a[-n:], b) for a, b in zip(big, small))
    del big, small, f
    x = x.view(-1, 64)[-(1 << 21) - 3:]                      # 2^21 tokens of 64, 2^32.5 hidden values
    ws = [torch.randn(2816, 64, device="cuda").bfloat16() / 8 for _ in range(2)] + [torch.randn(64, 2816, device="cuda").bfloat16() / 50]
    with torch.no_grad():
        y = gated_ffn(x, *ws)
        assert torch.equal(y[-n:], gated_ffn(x[-n:], *ws))


def test_gradients_past_32_bits():
    """The backward's offsets too: gradients of the last rows, and the weight's from them alone."""
    from dsalt import gated_ffn
    T, n = (1 << 20) + 37, 500
    x = torch.zeros(T, 64, device="cuda", dtype=torch.bfloat16)
    x[-n:] = torch.randn(n, 64, device="cuda")
    ws = [torch.randn(s, device="cuda").bfloat16() / 8 for s in ((4224, 64), (4224, 64), (64, 4224))]
    dy = torch.zeros(T, 64, device="cuda", dtype=torch.bfloat16)
    dy[-n:] = torch.randn(n, 64, device="cuda")

    def grads(x, dy):
        ts = [t.detach().requires_grad_(True) for t in (x, *ws)]
        return torch.autograd.grad(gated_ffn(*ts), ts, dy)

    big, small = grads(x, dy), grads(x[-n:], dy[-n:])
    assert torch.equal(big[0][-n:], small[0]) and not big[0][:-n].any()
    for a, b in zip(big[1:], small[1:]):  # the same terms at other places of the fp32 sum, one rounding
        mag = b.float().abs().max()
        assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 2.0 ** -10 * mag).all()
