"""The conditioning operators as a block uses them one after the other, and the model code that calls them."""
import pytest
import torch

from telefuser_b200.models import liveact_dit as LA
from telefuser_b200.models import longcat_video_dit as LC
from telefuser_b200.models import ltx_dit as LTX
from telefuser_b200.ops import context_attention as CA
from telefuser_b200.ops import functional as TF


def block(x, states, lens, clip, w, mods):
    """Cross attention to padded text between two norms, then attention over a cached clip and the block's own tokens."""
    H, D = 4, 64
    gate, shift, scale = mods
    h = TF.rmsnorm_modulate(x, w["n0"], shift, scale)
    q = TF.linear(h, w["q"]).unflatten(-1, (H, D))
    kv = TF.linear(states, w["kv"])
    k, v = kv[..., : H * D].unflatten(-1, (H, D)), kv[..., H * D :].unflatten(-1, (H, D))
    a = TF.linear(CA.cross_attention(q, k, v, kv_lens=lens).flatten(-2), w["o"])
    x, h = TF.rmsnorm_gate_residual_modulate(x, a, w["n1"], gate, w["n2"], shift, scale)
    q, k, v = (TF.linear(h, w[n]).unflatten(-1, (H, D)) for n in ("q", "k2", "v2"))
    a = TF.linear(CA.prefix_attention(q, clip[0], clip[1], k, v).flatten(-2), w["o"])
    return TF.rmsnorm_gate_residual_modulate(x, a, w["n1"], gate, w["n2"], shift, scale)


def inputs(device, dtype, B=2, S=200, L=77, P=150, C=256):
    g = torch.Generator(device="cpu").manual_seed(0)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std)  # noqa: E731
    w = {n: r(C, C, std=C**-0.5) for n in ("q", "o", "k2", "v2")} | {"kv": r(2 * C, C, std=C**-0.5)}
    w |= {n: 1 + r(C, std=0.1) for n in ("n0", "n1", "n2")}
    w = {n: t.to(device, dtype) for n, t in w.items()}
    mods = [r(B, 1, C, std=0.3).to(device) for _ in range(3)]
    clip = [r(1, P, 4, 64).to(device, dtype) for _ in range(2)]
    lens = torch.tensor([L, 11], dtype=torch.int32, device=device)
    return r(B, S, C).to(device, dtype), r(B, L, C).to(device, dtype), lens, clip, w, mods


def test_block_runs_on_cpu_and_padding_does_not_matter():
    x, states, lens, clip, w, mods = inputs("cpu", torch.float32)
    out = block(x, states, lens, clip, w, mods)
    states[1, 11:] = 1e4
    again = block(x, states, lens, clip, w, mods)
    assert all(torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 8, 200, 1000])
def test_block_matches_its_fp32_evaluation(S):
    """bf16 kernels against the same chain in fp32. Every stage rounds its output by at most 2^-8 of it (linear, norm, attention;
    P once more), about ten stages lie in a row with gains near one, so 2 % of the norm is twice their plain sum of
    relative half steps taken as independent (10^0.5 x 2^-8 = 1.2 %)."""
    x, states, lens, clip, w, mods = inputs("cuda", torch.bfloat16, S=S)
    got = block(x, states, lens, clip, w, mods)
    up = lambda t: t.float()  # noqa: E731
    TF.set_force_reference(True)
    try:
        want = block(up(x), up(states), lens, [up(t) for t in clip], {n: up(t) for n, t in w.items()}, mods)
    finally:
        TF.set_force_reference(False)
    for a, b in zip(got, want):
        assert ((a.float() - b).norm() / b.norm()).item() < 0.02


def test_longcat_text_attention_takes_lengths_and_offsets():
    torch.manual_seed(0)
    m = LC.MultiHeadCrossAttention(32, 4)
    x, cond = torch.randn(3, 5, 32), torch.randn(1, 9, 32)
    lens = [4, 0, 5]
    out = m(x, cond, lens)
    assert torch.equal(out, m(x, cond, LC.text_offsets(lens, "cpu")))
    torch.testing.assert_close(out[2:], m(x[2:], cond[:, 4:], [5]))
    assert (out[1] == 0).all()


def test_longcat_cached_clip_is_shared_by_the_batch():
    torch.manual_seed(0)
    m = LC.Attention(32, 4)
    x = torch.randn(2, 6, 32)
    rope = (torch.ones(6, 4), torch.zeros(6, 4))
    cache = tuple(torch.randn(1, 7, 4, 8) for _ in range(2))
    out, _ = m(x, rope, kv_cache=cache)
    want, _ = m(x, rope, kv_cache=tuple(c.expand(2, -1, -1, -1) for c in cache))
    torch.testing.assert_close(out, want)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_ltx_key_masks_equal_the_additive_mask(device):
    """One sample padded on the left, one full, one without any context token (which attends evenly)."""
    g = torch.Generator().manual_seed(0)
    dt = torch.bfloat16 if device == "cuda" else torch.float32
    q, k, v = (torch.randn(3, n, 2, 16, generator=g).to(device, dt) for n in (70, 40, 40))
    visible = torch.ones(3, 40, dtype=torch.bool, device=device)
    visible[0, :33] = False
    visible[2] = False
    additive = (visible.float() - 1)[:, None, None] * torch.finfo(torch.float32).max
    got, want = LTX._key_masked_attention(q, k, v, visible), LTX._masked_attention(q, k, v, additive)
    # both round the output (2^-8 of it in bf16), and the weights of the kernel's second product 2^-8 of sum p |v| <= max |v|
    tol = 2 * 2.0**-8 * v.float().abs().max().item() if device == "cuda" else 1e-5
    assert ((got.float() - want.float()).abs() <= tol + (2.0**-7 if device == "cuda" else 0) * want.float().abs()).all()


# ---- LTX context masks through the model ------------------------------------------------------------------------------
def ltx_model_and_inputs(B, S, adaln):
    torch.manual_seed(0)
    m = LTX.LTXModel(model_type=LTX.LTXModelType.VideoOnly, num_attention_heads=2, attention_head_dim=24, in_channels=8,
                     out_channels=8, num_layers=2, cross_attention_dim=48, rope_type=LTX.LTXRopeType.SPLIT,
                     cross_attention_adaln=adaln)  # fmt: skip
    for p in m.parameters():
        torch.nn.init.normal_(p, std=0.2)
    T = 6
    start = torch.arange(T, dtype=torch.float32)[None, None].expand(B, 3, T)
    sigma = torch.linspace(0.9, 0.4, B)
    return m.float().eval(), dict(latent=torch.randn(B, T, 8), sigma=sigma, positions=torch.stack([start, start + 1], dim=-1),
                                  timesteps=sigma[:, None].expand(B, T), context=torch.randn(B, S, 48))  # fmt: skip


@pytest.mark.parametrize("adaln", [False, True])
@pytest.mark.parametrize("B,mask", [
    (2, [[0, 0, 1, 1, 1, 0, 1]]),  # one mask for all samples
    (2, [[0, 0, 1, 1, 1, 0, 1], [1, 1, 1, 1, 0, 0, 0]]),
    (2, [[0, 0, 0, 0, 0, 0, 0], [1, 0, 0, 0, 0, 0, 0]]),  # a sample without a token
    (2, [[0, 0, 0, 0, 0, 0, 0]]),
    (1, [[1, 0, 1, 0, 1, 0, 1]]),
    (3, [[0, 1, 1, 1, 1, 1, 1]]),
])  # fmt: skip
@pytest.mark.parametrize("shape", ["rows", "unit axis", "two unit axes", "bool"])
def test_ltx_model_context_masks_equal_the_additive_form(B, mask, shape, adaln):
    m, kw = ltx_model_and_inputs(B, 7, adaln)
    ones = torch.tensor(mask)
    additive = (ones.float() - 1)[:, None, None] * torch.finfo(torch.float32).max
    ones = {"rows": ones, "unit axis": ones[:, None], "two unit axes": ones[:, None, None], "bool": ones.bool()}[shape]
    want, _ = m(LTX.Modality(context_mask=additive, **kw), None)
    got, _ = m(LTX.Modality(context_mask=ones, **kw), None)
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4)
    if B > 1 and mask != [[0] * 7]:
        assert not torch.allclose(got, m(LTX.Modality(context_mask=None, **kw), None)[0], atol=1e-3)


def test_ltx_model_context_mask_per_query_stays_additive():
    m, kw = ltx_model_and_inputs(2, 7, False)
    marks = torch.ones(1, 6, 7, dtype=torch.int64)
    marks[0, 2:, 3:] = 0
    want, _ = m(LTX.Modality(context_mask=(marks.float() - 1)[:, None] * torch.finfo(torch.float32).max, **kw), None)
    torch.testing.assert_close(m(LTX.Modality(context_mask=marks, **kw), None)[0], want)


@pytest.mark.parametrize("B", [1, 2])
@pytest.mark.parametrize("kept,running", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.float64, torch.float32)])
def test_longcat_cached_clip_of_another_type(B, kept, running):
    """Keys that were kept in one type under a model that runs in another join in the wider of the two."""
    torch.manual_seed(0)
    m = LC.Attention(32, 4).to(running)
    x = torch.randn(B, 6, 32).to(running)
    rope = (torch.ones(6, 4), torch.zeros(6, 4))
    cache = tuple(torch.randn(1, 7, 4, 8).to(kept) for _ in range(2))
    got, _ = m(x, rope, kv_cache=cache)
    want, _ = m(x, rope, kv_cache=tuple(c.to(torch.promote_types(kept, running)).expand(B, -1, -1, -1).clone() for c in cache))
    assert got.dtype == running
    u = torch.finfo(running).eps  # both round their output once, from evaluations in fp32 of the same values
    torch.testing.assert_close(got, want, rtol=u, atol=1e-5 if running == torch.float32 else u)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 2])
def test_longcat_cached_clip_of_another_type_on_gpu(B):
    torch.manual_seed(0)
    m = LC.Attention(256, 2).to("cuda", torch.bfloat16)
    x = torch.randn(B, 70, 256, device="cuda", dtype=torch.bfloat16)
    rope = (torch.ones(70, 64, device="cuda"), torch.zeros(70, 64, device="cuda"))
    cache = tuple(torch.randn(1, 90, 2, 128, device="cuda") for _ in range(2))
    got, _ = m(x, rope, kv_cache=cache)
    assert torch.equal(got, m(x, rope, kv_cache=tuple(c.bfloat16() for c in cache))[0])


def test_longcat_text_lengths_as_a_tensor():
    torch.manual_seed(0)
    m = LC.MultiHeadCrossAttention(32, 4)
    x, cond = torch.randn(3, 5, 32), torch.randn(1, 9, 32)
    want = m(x, cond, [4, 0, 5])
    assert torch.equal(m(x, cond, torch.tensor([4, 0, 5])), want)
    assert torch.equal(m(x, cond, (4, 0, 5, 7)), want)  # one length per sample is looked at
    assert LC.text_offsets([4, 0, 5], "cpu").tolist() == LC.text_offsets(torch.tensor([4, 0, 5]), "cpu").tolist() == [0, 4, 4, 9]


@pytest.mark.gpu
def test_longcat_text_attention_in_a_captured_graph():
    """Lengths given as numbers need no copy from the host, so the call can be captured."""
    torch.manual_seed(0)
    m = LC.MultiHeadCrossAttention(256, 2).to("cuda", torch.bfloat16)
    x, cond = torch.randn(2, 70, 256, device="cuda").bfloat16(), torch.randn(1, 30, 256, device="cuda").bfloat16()
    with torch.no_grad():
        want = m(x, cond, [19, 11])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = m(x, cond, [19, 11])
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("B,n_t", [(1, 3), (2, 1), (2, 3)])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_liveact_one_audio_window_serves_every_frame(B, n_t, device):
    torch.manual_seed(0)
    dt = torch.bfloat16 if device == "cuda" else torch.float32
    m = LA.SingleStreamAttention(64, 48, 4).to(device, dt)
    x, enc = torch.randn(B, n_t * 6, 64).to(device, dt), torch.randn(1, 4, 5, 48).to(device, dt)
    got = m(x, enc, (n_t, 2, 3), start_f=3)  # only the last window is left
    frames = x.reshape(B * n_t, 6, 64)
    want = torch.cat([m(f[None], enc[:, 3:], (1, 2, 3)) for f in frames]).reshape(B, n_t * 6, 64)
    torch.testing.assert_close(got, want, rtol=torch.finfo(dt).eps, atol=torch.finfo(dt).eps)
