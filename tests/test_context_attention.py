"""Context attention (`cross_attention`, `prefix_attention`) against the definition in 64 bits."""
import math

import pytest
import torch

from telefuser_b200.ops import context_attention as CA
from telefuser_b200.ops import functional as TF
from telefuser_b200.ops import native

BF, FP = torch.bfloat16, torch.float16


def exact(q, keys, scale=None):
    """q [B, Sq, H, D]; keys: per sample the (k [n, Hkv, D], v) that it sees. -> out, lse, sum p |v|, sum |v|, the largest
    sum |q_d k_d| scale, all in 64 bits."""
    B, Sq, H, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Sq, H, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, H, Sq), float("-inf"), dtype=torch.float64, device=q.device)
    pv, sv = torch.zeros_like(out), torch.zeros_like(out)
    size = 0.0
    for b, (k, v) in enumerate(keys):
        if k.shape[0] == 0 or Sq == 0:
            continue
        G = H // k.shape[1]
        kd, vd = (t.double().repeat_interleave(G, dim=1) for t in (k, v))
        qd = q[b].double()
        s = torch.einsum("ihd,jhd->hij", qd, kd) * scale
        size = max(size, (torch.einsum("ihd,jhd->hij", qd.abs(), kd.abs()) * scale).max().item())
        p = torch.softmax(s, dim=-1)
        lse[b] = torch.logsumexp(s, dim=-1)
        out[b] = torch.einsum("hij,jhd->ihd", p, vd)
        pv[b] = torch.einsum("hij,jhd->ihd", p, vd.abs())
        sv[b] = vd.abs().sum(0)
    return out, lse, pv, sv, size


def check(got, lse, want, dtype):
    """Roundings counted: the output's (half a step of the type, u), each weight's on its way into the second product (u, or
    2^-25 of the largest where fp16 has no normal number left), and the fp32 scores, their exponentials and sums: a product
    of D <= 128 terms, its scaling and ex2 leave a score off by at most 2^-17 of sum |q_d k_d| scale, and a weight by that
    and a few 2^-22, on both sides of the quotient."""
    out, lse64, pv, sv, size = want
    u = torch.finfo(dtype).eps / 2
    eps = 2.0**-17 * (1 + size)
    tol = u * out.abs() + (u + 2 * eps) * (1 + u) * pv + (2.0**-25 * sv if dtype == FP else 0)
    err = (got.double() - out).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {(err / tol.clamp_min(1e-300)).max().item():.2f} of the tolerance"
    if lse is not None:
        empty = lse64 == float("-inf")
        assert (lse[empty] == float("-inf")).all() and torch.isfinite(lse[~empty]).all()
        assert ((lse.double() - lse64)[~empty].abs() <= eps + 2.0**-20 * lse64[~empty].abs()).all()


def rand(g, *shape, dtype, device, std=1.0):
    return (torch.randn(*shape, generator=g, device=device) * std).to(dtype)


def make(B, Sq, H, Hkv, D, Skv, dtype, device, seed=0, std=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    q = rand(g, B, Sq, H, D, dtype=dtype, device=device, std=std)
    k = rand(g, B, Skv, Hkv, D, dtype=dtype, device=device, std=std)
    v = rand(g, B, Skv, Hkv, D, dtype=dtype, device=device) + 0.5
    return q, k, v


def poison(t, visible):
    """Infinities and NaN in every place that `visible` [B, Skv] hides."""
    t = t.clone()
    bad = torch.tensor([float("nan"), float("inf"), float("-inf")], device=t.device, dtype=t.dtype)
    fill = bad[torch.arange(t.shape[1], device=t.device) % 3][None, :, None, None].expand_as(t)
    return torch.where(visible[:, :, None, None], t, fill)


def pick(k, v, visible):
    return [(k[b, visible[b]], v[b, visible[b]]) for b in range(k.shape[0])]


# ---- CPU: semantics and refusals --------------------------------------------------------------------------------------
def test_reference_forms_agree_on_cpu():
    q, k, v = make(3, 5, 4, 2, 16, 9, torch.float32, "cpu")
    lens = [9, 0, 4]
    visible = torch.arange(9)[None] < torch.tensor(lens)[:, None]
    o, lse = CA.cross_attention(q, poison(k, visible), poison(v, visible), kv_lens=lens, return_lse=True)
    out, lse64, *_ = exact(q, pick(k, v, visible))
    torch.testing.assert_close(o.double(), out, rtol=1e-5, atol=1e-5)
    assert (o[1] == 0).all() and (lse[1] == float("-inf")).all()
    torch.testing.assert_close(lse.double(), lse64, rtol=1e-5, atol=1e-5)
    masked = CA.cross_attention(q, k, v, key_mask=visible)
    torch.testing.assert_close(masked, o)
    kp, vp = k[visible], v[visible]
    cu = [0, 9, 9, 13]
    torch.testing.assert_close(CA.cross_attention(q, kp, vp, cu_kv=cu), o)
    torch.testing.assert_close(CA.cross_attention(q, kp[None], vp[None], cu_kv=torch.tensor(cu)), o)
    blocks = CA.context_attention_reference(q, k, v, visible, q_block=2)
    torch.testing.assert_close(blocks, o)


def test_prefix_equals_concatenation_on_cpu():
    q, k, v = make(2, 3, 4, 4, 8, 6, torch.float32, "cpu")
    _, kp, vp = make(1, 1, 4, 4, 8, 11, torch.float32, "cpu", seed=1)
    cat = lambda a, b: torch.cat([a.expand(2, -1, -1, -1), b], dim=1)  # noqa: E731
    torch.testing.assert_close(CA.prefix_attention(q, kp, vp, k, v), TF.attention(q, cat(kp, k), cat(vp, v)))
    o, lse = CA.prefix_attention(q, kp[0], vp[0], k, v, kv_lens=[6, 0], return_lse=True)
    want, wl = TF.attention(q[1:], kp, vp, return_lse=True)
    torch.testing.assert_close(o[1:], want)
    torch.testing.assert_close(lse[1:], wl)


@pytest.mark.parametrize("call", [
    lambda q, k, v: CA.cross_attention(q[0], k, v),
    lambda q, k, v: CA.cross_attention(q, k, v[:, :-1]),
    lambda q, k, v: CA.cross_attention(q[:, :, :3], k, v),
    lambda q, k, v: CA.cross_attention(q, k.double(), v),
    lambda q, k, v: CA.cross_attention(q[:1], k, v),
    lambda q, k, v: CA.cross_attention(q, k, v, kv_lens=[1]),
    lambda q, k, v: CA.cross_attention(q, k, v, kv_lens=[1, 8]),
    lambda q, k, v: CA.cross_attention(q, k, v, kv_lens=[-1, 1]),
    lambda q, k, v: CA.cross_attention(q, k, v, key_mask=torch.ones(2, 6, dtype=torch.bool)),
    lambda q, k, v: CA.cross_attention(q, k, v, key_mask=torch.ones(2, 7)),
    lambda q, k, v: CA.cross_attention(q, k, v, cu_kv=[0, 3, 7]),
    lambda q, k, v: CA.cross_attention(q, k[0], v[0], cu_kv=[0, 7]),
    lambda q, k, v: CA.cross_attention(q, k[0], v[0], cu_kv=[0, 5, 3]),
    lambda q, k, v: CA.cross_attention(q, k[0], v[0], cu_kv=[0, 3, 8]),
    lambda q, k, v: CA.cross_attention(q, k[0], v[0], cu_kv=[0, 3, 7], kv_lens=[1, 1]),
    lambda q, k, v: CA.cross_attention(q, k, v, scale=0.0),
    lambda q, k, v: CA.cross_attention(q, k, v, scale=-1.0),
    lambda q, k, v: CA.cross_attention(q, k, v, scale=float("nan")),
    lambda q, k, v: CA.prefix_attention(q, k, v, k, v),
    lambda q, k, v: CA.prefix_attention(q, k[:1, :, :1], v[:1, :, :1], k, v),
    lambda q, k, v: CA.prefix_attention(q, k[:1], v[:1], k[:1], v[:1]),
    lambda q, k, v: CA.prefix_attention(q, k[:1], v[:1], k, v, kv_lens=[0, 8]),
])  # fmt: skip
def test_refusals(call):
    q, k, v = make(2, 3, 4, 2, 8, 7, torch.float32, "cpu")
    with pytest.raises(ValueError):
        call(q, k, v)


# ---- GPU --------------------------------------------------------------------------------------------------------------
gpu = pytest.mark.gpu


@pytest.fixture
def lib():
    native.load()
    yield
    torch.cuda.synchronize()
    assert native.last_status() == 0


def _lens(B, Skv, least=0):
    return [Skv] if B == 1 else [least + (Skv - least) * ((b * 3 + 1) % B) // (B - 1) for b in range(B)]


ROWS = [  # few query rows: single tokens, grouped heads, one to many keys
    (1, 1, 1, 1, 64, 1), (2, 1, 4, 4, 128, 17), (3, 1, 8, 1, 128, 300), (2, 4, 8, 2, 64, 1000), (5, 16, 3, 3, 128, 129),
    (1, 2, 6, 2, 72, 4097), (2, 1, 16, 1, 40, 33), (4, 3, 10, 2, 8, 95), (1, 1, 2, 2, 128, 40000),
]
TILES = [  # query tiles: one tile, two, odd numbers, grouped heads that share a tile or do not
    (1, 17, 1, 1, 128, 1), (2, 128, 2, 2, 128, 128), (2, 129, 2, 1, 64, 257), (3, 300, 3, 1, 128, 77), (1, 64, 8, 1, 128, 515),
    (2, 257, 4, 4, 96, 512), (2, 31, 32, 1, 64, 33), (1, 1000, 2, 2, 40, 640), (4, 20, 6, 2, 128, 1100), (1, 130, 1, 1, 128, 9000),
]
SHORT = [  # many query rows, at most 64 keys
    (2, 40, 1, 1, 128, 1), (3, 1000, 3, 1, 64, 32), (2, 333, 4, 2, 128, 64), (2, 100, 10, 2, 72, 17), (1, 5000, 2, 2, 40, 63),
    (9, 65, 16, 4, 128, 50),
]


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("shape", ROWS + TILES + SHORT)
def test_dense(lib, shape, dtype):
    q, k, v = make(*shape, dtype, "cuda")
    o, lse = CA.cross_attention(q, k, v, return_lse=True)
    check(o, lse, exact(q, [(k[b], v[b]) for b in range(q.shape[0])]), dtype)


@gpu
@pytest.mark.parametrize("shape", ROWS + TILES + SHORT)
@pytest.mark.parametrize("layout", ["padded", "packed", "masked", "masked_lens"])
def test_lengths_and_masks(lib, shape, layout):
    """Ragged samples, one of them empty; what is hidden holds NaN and infinities."""
    B, Sq, H, Hkv, D, Skv = shape
    q, k, v = make(*shape, BF, "cuda", seed=1)
    lens = torch.tensor(_lens(B, Skv), device="cuda")
    visible = torch.arange(Skv, device="cuda")[None] < lens[:, None]
    if layout.startswith("masked"):
        g = torch.Generator(device="cuda").manual_seed(2)
        holes = torch.rand(B, Skv, generator=g, device="cuda") < 0.5
        holes[:, : Skv // 2] |= (torch.arange(Skv // 2, device="cuda") // 128 % 2 == 0)[None]  # whole blocks of nothing
        mask = ~holes
        visible = mask if layout == "masked" else mask & visible
    want = exact(q, pick(k, v, visible))
    kx, vx = poison(k, visible), poison(v, visible)
    if layout == "packed":
        edge = torch.full((3, Hkv, D), float("nan"), device="cuda", dtype=BF)  # rows behind the last sample
        kx, vx = torch.cat([k[visible], edge]), torch.cat([v[visible], edge])
        cu = torch.cat([lens.new_zeros(1), lens.cumsum(0)]).to(torch.int32)
        o, lse = CA.cross_attention(q, kx, vx, cu_kv=cu, return_lse=True)
    elif layout == "padded":
        o, lse = CA.cross_attention(q, kx, vx, kv_lens=lens, return_lse=True)
    else:
        o, lse = CA.cross_attention(q, kx, vx, kv_lens=lens if layout == "masked_lens" else None, key_mask=mask, return_lse=True)
    check(o, lse, want, BF)
    none = ~visible.any(1)
    assert (o[none] == 0).all() and (lse[none] == float("-inf")).all()


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("shape,P", [
    ((1, 1, 1, 1, 64, 1), 1), ((3, 4, 8, 2, 64, 33), 77), ((64, 1, 8, 2, 128, 100), 1000), ((5, 1, 4, 4, 128, 1), 3000),
    ((2, 7, 6, 2, 128, 65), 130), ((2, 300, 2, 2, 128, 129), 257), ((2, 128, 4, 1, 64, 200), 64), ((1, 500, 2, 1, 96, 77), 600),
    ((3, 40, 2, 2, 128, 0), 100), ((20, 2, 4, 2, 64, 70), 9000), ((9, 1, 24, 8, 128, 20), 2500), ((3, 2, 2, 2, 128, 50), 0), ((2, 200, 2, 2, 128, 50), 0), ((2, 200, 2, 2, 128, 0), 50),
])  # fmt: skip
@pytest.mark.parametrize("ragged", [False, True])
def test_prefix(lib, shape, P, ragged, dtype):
    B, Sq, H, Hkv, D, S = shape
    q, k, v = make(*shape, dtype, "cuda", seed=3)
    _, kp, vp = make(1, 1, 1, Hkv, D, P, dtype, "cuda", seed=4)
    lens = _lens(B, S) if ragged else [S] * B
    visible = torch.arange(S, device="cuda")[None] < torch.tensor(lens, device="cuda")[:, None]
    keys = [(torch.cat([kp[0], a]), torch.cat([vp[0], b])) for a, b in pick(k, v, visible)]
    o, lse = CA.prefix_attention(q, kp, vp, poison(k, visible), poison(v, visible), kv_lens=lens if ragged else None,
                                 return_lse=True)  # fmt: skip
    check(o, lse, exact(q, keys), dtype)


@gpu
@pytest.mark.parametrize("Sq", [2, 200])
def test_strided_views_and_head_major_states(lib, Sq):
    """q as a slice of a fused projection, k / v as slices of another, and states stored [B, H, S, D]."""
    B, H, D, Skv = 2, 4, 128, 150
    g = torch.Generator(device="cuda").manual_seed(5)
    fused = rand(g, B, Sq, 3 * H * D, dtype=BF, device="cuda")
    kv = rand(g, B, Skv, 2 * H * D, dtype=BF, device="cuda")
    q = fused[..., H * D : 2 * H * D].unflatten(-1, (H, D))
    k, v = kv[..., : H * D].unflatten(-1, (H, D)), kv[..., H * D :].unflatten(-1, (H, D))
    want = exact(q, [(k[b], v[b]) for b in range(B)])
    check(*CA.cross_attention(q, k, v, return_lse=True), want, BF)
    km, vm = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    check(*CA.cross_attention(q, km, vm, return_lse=True), want, BF)
    odd = torch.empty(k.numel() + 1, device="cuda", dtype=BF)[1:].view(k.shape).copy_(k)  # base not on 16 bytes
    check(*CA.cross_attention(q, odd, v, return_lse=True), want, BF)
    one = CA.cross_attention(q, k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1))
    check(one, None, exact(q, [(k[0], v[0])] * B), BF)
    _, kp, vp = make(1, 1, 1, H, D, 70, BF, "cuda", seed=6)
    keys = [(torch.cat([kp[0], k[b]]), torch.cat([vp[0], v[b]])) for b in range(B)]
    check(*CA.prefix_attention(q, kp, vp, k, v, return_lse=True), exact(q, keys), BF)
    check(*CA.prefix_attention(q[:, ::2], kp, vp, k, v, return_lse=True), exact(q[:, ::2], keys), BF)


@gpu
@pytest.mark.parametrize("Sq", [1, 140])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_peaked_scores_and_scale(lib, Sq, dtype):
    """Maxima that keep growing along the keys (the rescale path) and a scale of the caller's."""
    q, k, v = make(2, Sq, 2, 2, 128, 1000, dtype, "cuda", seed=7)
    k = (k * torch.linspace(0.1, 6.0, 1000, device="cuda")[None, :, None, None]).to(dtype)
    check(*CA.cross_attention(q, k, v, scale=0.2, return_lse=True), exact(q, [(k[b], v[b]) for b in range(2)], 0.2), dtype)



@gpu
@pytest.mark.parametrize("layout", ["padded", "packed", "masked"])
def test_long_runs_of_tiles_without_keys(lib, layout):
    """Samples without states among others, each of them several tiles per SM, with one and with three blocks of keys."""
    B, Sq, H, D = 4, 24001, 8, 64
    lens = [300, 0, 0, 90]
    q, k, v = make(B, Sq, H, H, D, 300, BF, "cuda", seed=11)
    visible = torch.arange(300, device="cuda")[None] < torch.tensor(lens, device="cuda")[:, None]
    if layout == "packed":
        o, lse = CA.cross_attention(q, k[visible], v[visible], cu_kv=[0, 300, 300, 300, 390], return_lse=True)
    elif layout == "padded":
        o, lse = CA.cross_attention(q, k, v, kv_lens=lens, return_lse=True)
    else:
        o, lse = CA.cross_attention(q, k, v, key_mask=visible, return_lse=True)
    check(o, lse, exact(q, pick(k, v, visible)), BF)
    assert (o[1:3] == 0).all() and (lse[1:3] == float("-inf")).all()


@gpu
@pytest.mark.parametrize("Sq", [2, 130])
def test_device_lengths_out_of_range_are_clamped(lib, Sq):
    q, k, v = make(3, Sq, 2, 2, 64, 90, BF, "cuda", seed=8)
    wild = torch.tensor([-5, 1 << 30, 60], dtype=torch.int64, device="cuda")
    same = CA.cross_attention(q, k, v, kv_lens=[0, 90, 60])
    assert torch.equal(CA.cross_attention(q, k, v, kv_lens=wild), same)
    kp, vp = k.reshape(-1, 2, 64), v.reshape(-1, 2, 64)
    cu = torch.tensor([-7, 100, 50, 1 << 20], dtype=torch.int32, device="cuda")
    o = CA.cross_attention(q, kp, vp, cu_kv=cu)
    check(o, None, exact(q, [(kp[:100], vp[:100]), (kp[:0], vp[:0]), (kp[50:], vp[50:])]), BF)


@gpu
def test_no_queries_and_no_states(lib):
    q, k, v = make(2, 0, 2, 2, 64, 9, BF, "cuda")
    assert CA.cross_attention(q, k, v).shape == (2, 0, 2, 64)
    for Sq in (1, 200):
        q, k, v = make(2, Sq, 2, 2, 64, 0, BF, "cuda")
        o, lse = CA.cross_attention(q, k, v, return_lse=True)
        assert (o == 0).all() and (lse == float("-inf")).all()


@gpu
def test_other_types_and_head_dims_take_the_fp32_evaluation(lib):
    q, k, v = make(2, 6, 2, 1, 20, 11, BF, "cuda")
    check(CA.cross_attention(q, k, v), None, exact(q, [(k[b], v[b]) for b in range(2)]), BF)
    q, k, v = make(2, 6, 2, 1, 160, 11, torch.float32, "cuda")
    o = CA.cross_attention(q, k, v, kv_lens=torch.tensor([4, 11], device="cuda"))
    torch.testing.assert_close(o.double(), exact(q, [(k[0, :4], v[0, :4]), (k[1], v[1])])[0], rtol=1e-4, atol=1e-4)


@gpu
@pytest.mark.parametrize("Sq,Skv", [(1, 5000), (300, 700), (20, 9000)])
def test_same_bits_again_on_another_stream_and_replayed(lib, Sq, Skv):
    """Results do not depend on the run, the stream or a capture; two captured graphs do not share scratch."""
    q, k, v = make(2, Sq, 8, 2, 128, Skv, BF, "cuda", seed=9)
    _, kp, vp = make(1, 1, 1, 2, 128, 500, BF, "cuda", seed=10)
    lens = torch.tensor([Skv, Skv // 3], dtype=torch.int32, device="cuda")
    first = [CA.cross_attention(q, k, v, kv_lens=lens), CA.prefix_attention(q, kp, vp, k, v, kv_lens=lens)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [CA.cross_attention(q, k, v, kv_lens=lens), CA.prefix_attention(q, kp, vp, k, v, kv_lens=lens)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    with torch.cuda.graph(graphs[0]):
        outs.append(CA.cross_attention(q, k, v, kv_lens=lens))
    with torch.cuda.graph(graphs[1]):
        outs.append(CA.prefix_attention(q, kp, vp, k, v, kv_lens=lens))
    lens.copy_(torch.tensor([7, Skv], device="cuda"))
    graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    now = [CA.cross_attention(q, k, v, kv_lens=lens), CA.prefix_attention(q, kp, vp, k, v, kv_lens=lens)]
    assert all(torch.equal(a, b) for a, b in zip(outs, now))


@gpu
@pytest.mark.parametrize("fp16", [False, True])
def test_first_block_arrives_last(lib, fp16):
    """The tile kernel's first K tile comes from memory while the second block and the first V tile are in L2, so the load of
    its first stage is the slowest; the keys end inside the second block, behind NaN."""
    dtype = FP if fp16 else BF
    B, Sq, H, D, Skv, n = 148, 40, 1, 128, 256, 177
    q, k, v = make(B, Sq, H, H, D, Skv, dtype, "cuda", seed=12)
    visible = (torch.arange(Skv, device="cuda") < n).expand(B, -1)
    k, v = poison(k, visible), poison(v, visible)
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    want = exact(q, pick(k, v, visible))
    flush = torch.empty(64 << 20, device="cuda", dtype=torch.float32)  # twice the L2 cache
    for _ in range(20):
        flush.fill_(1.0)
        (k[:, 128:].isnan().sum() + v[:, :128].isnan().sum() + q.isnan().sum())
        o, lse = CA.cross_attention(q, k, v, kv_lens=lens, return_lse=True)
        check(o, lse, want, dtype)


# ---- NaN and infinities among the keys that are seen ------------------------------------------------------------------
SPECIAL = [  # rows kernel without and with a key split, tile kernel without and with one, short kernel
    (2, 1, 4, 2, 64, 300), (1, 1, 2, 1, 128, 9000), (3, 5, 4, 4, 64, 33), (2, 300, 2, 1, 64, 400), (1, 60, 1, 1, 128, 4000),
    (1, 200, 2, 2, 128, 2000), (2, 100, 4, 2, 128, 50), (2, 70, 2, 2, 40, 17),
]


def special(t, at, value):
    t = t.clone()
    t[at] = value
    return t


def same_kind(got, lse, o64, lse64):
    """NaN where the definition in 64 bits has NaN, the infinities that it has, and finite values elsewhere."""
    for a, b in ((got, o64), (lse, lse64)):
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.double().masked_fill(~a.isinf(), 0), b.masked_fill(~b.isinf(), 0))


def special_cases(q, k, v):
    nan, inf = float("nan"), float("inf")
    last = k.shape[1] - 1
    yield "nan in a key", q, special(k, (0, last // 2, 0, 3), nan), v
    yield "nan in the first key", q, special(k, (0, 0, 0, 3), nan), v
    yield "inf in a key", q, special(k, (0, last, -1, 0), inf), v
    yield "-inf in a key", q, special(k, (0, last // 3, 0, 1), -inf), v
    yield "inf and nan in keys", q, special(special(k, (0, last, 0, 0), inf), (0, 0, 0, 1), nan), v
    yield "nan in a value", q, k, special(v, (0, last // 2, 0, 3), nan)
    yield "inf in a value", q, k, special(v, (0, last, 0, 2), inf)
    yield "nan in a query", special(q, (0, q.shape[1] - 1, 0, 5), nan), k, v
    yield "inf in a query", special(q, (-1, 0, -1, 5), inf), k, v
    yield "every key -inf", q.abs(), special(k, (0, slice(None), 0), -inf), v
    yield "every key -inf, nan in a value", q.abs(), special(k, (0, slice(None), 0), -inf), special(v, (0, last // 2, 0, 3), nan)


def definition(q, keys, scale=None):
    """`exact` with what infinities and NaN do in the sums, as the fp32 evaluation has it: a query whose scores are all -inf
    has weights of zero."""
    B, Sq, H, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Sq, H, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, H, Sq), float("-inf"), dtype=torch.float64, device=q.device)
    for b, (k, v) in enumerate(keys):
        kd, vd = (t.double().repeat_interleave(H // k.shape[1], dim=1).transpose(0, 1) for t in (k, v))
        s = q[b].double().transpose(0, 1) @ kd.transpose(1, 2) * scale
        lse[b] = torch.logsumexp(s, dim=-1)
        p = torch.exp(s - lse[b].masked_fill(lse[b] == float("-inf"), 0.0)[..., None])
        out[b] = (p @ vd).transpose(0, 1)
    return out, lse


def check_special(q, k, v, dtype):
    B = q.shape[0]
    for what, qx, kx, vx in special_cases(q, k, v):
        want = definition(qx, [(kx[b], vx[b]) for b in range(B)])
        o, lse = CA.cross_attention(qx, kx, vx, return_lse=True)
        try:
            same_kind(o, lse, *want)
        except AssertionError as e:
            raise AssertionError(what) from e
        # rows that come out finite have their values: a key at -inf weighs nothing
        fine = want[0].isfinite().all(-1)[..., None]
        _, _, pv, sv, _ = exact(qx, [(kx[b], vx[b]) for b in range(B)])
        size = exact(q, [(k[b], v[b]) for b in range(B)])[-1]  # finite scores are those of q and k
        zero = torch.zeros_like(want[0])
        check(torch.where(fine, o, torch.zeros_like(o)), None, (torch.where(fine, want[0], zero), None,
              pv.where(fine & pv.isfinite(), zero), sv.where(sv.isfinite(), zero), size), dtype)  # fmt: skip


@pytest.mark.parametrize("shape", SPECIAL)
def test_special_values_on_cpu(shape):
    q, k, v = make(*shape, torch.float32, "cpu", seed=13)
    B = q.shape[0]
    for what, qx, kx, vx in special_cases(q, k, v):
        o, lse = CA.cross_attention(qx, kx, vx, return_lse=True)
        same_kind(o, lse, *definition(qx, [(kx[b], vx[b]) for b in range(B)]))


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("shape", SPECIAL)
def test_special_values(lib, shape, dtype):
    check_special(*make(*shape, dtype, "cuda", seed=13), dtype)


@gpu
@pytest.mark.parametrize("shape,P", [((2, 1, 4, 2, 64, 40), 3000), ((40, 1, 4, 1, 128, 20), 9000), ((2, 130, 2, 2, 64, 90), 140)])
def test_special_values_in_a_shared_prefix(lib, shape, P):
    B, Sq, H, Hkv, D, S = shape
    q, k, v = make(*shape, BF, "cuda", seed=14)
    _, kp, vp = make(1, 1, 1, Hkv, D, P, BF, "cuda", seed=15)
    nan, inf = float("nan"), float("inf")
    for qx, kpx, vpx, kx, vx in [
        (q, special(kp, (0, P - 1, 0, 2), nan), vp, k, v), (q, kp, vp, special(k, (1, S - 1, 0, 2), nan), v),
        (special(q, (1, 0, 0, 0), nan), kp, vp, k, v), (q, special(kp, (0, 0, 0, 2), inf), vp, k, v),
        (q, kp, special(vp, (0, P // 2, 0, 1), nan), k, v), (q, kp, vp, k, special(v, (0, 0, 0, 1), nan)),
        (q, special(kp, (0, 1, 0, 2), inf), vp, special(k, (0, 0, 0, 1), nan), v),
    ]:  # fmt: skip
        o, lse = CA.prefix_attention(qx, kpx, vpx, kx, vx, return_lse=True)
        same_kind(o, lse, *definition(qx, [(torch.cat([kpx[0], kx[b]]), torch.cat([vpx[0], vx[b]])) for b in range(B)]))


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("B,Sq,H", [(0, 3, 4), (2, 0, 4), (2, 3, 0), (0, 0, 0)])
def test_empty_queries_give_empty_results(B, Sq, H, device, dtype):
    q, k, v = make(B, Sq, H, 2, 8, 5, dtype, device)
    _, kp, vp = make(1, 1, 1, 2, 8, 7, dtype, device)
    packed = [t.reshape(-1, 2, 8) for t in (k, v)]
    cu = torch.arange(B + 1, device=device) * 5
    for o, lse in [
        CA.cross_attention(q, k, v, return_lse=True), CA.cross_attention(q, k, v, kv_lens=[3] * B, return_lse=True),
        CA.cross_attention(q, k, v, key_mask=torch.ones(B, 5, dtype=torch.bool, device=device), return_lse=True),
        CA.cross_attention(q, *packed, cu_kv=cu, return_lse=True), CA.prefix_attention(q, kp, vp, k, v, return_lse=True),
    ]:  # fmt: skip
        assert o.shape == (B, Sq, H, 8) and o.dtype == dtype and lse.shape == (B, H, Sq) and lse.dtype == torch.float32


@pytest.mark.parametrize("scale", [1e39, 1e-39, 1e-60, float("inf"), 2.0**127.5])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_scales_beyond_fp32_are_refused(scale, device):
    q, k, v = make(2, 3, 4, 2, 8, 7, BF, device)
    with pytest.raises(ValueError, match="scale"):
        CA.cross_attention(q, k, v, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        CA.prefix_attention(q, k[:1], v[:1], k, v, scale=scale)


@pytest.mark.parametrize("lens", [[2.5, 3], torch.tensor([2.0, 3.25]), torch.tensor([[2], [3]]), torch.tensor([[2, 3]])])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_lengths_that_are_no_whole_numbers_are_refused(lens, device):
    q, k, v = make(2, 3, 4, 2, 8, 7, BF, device)
    with pytest.raises(ValueError):
        CA.cross_attention(q, k, v, kv_lens=lens)
    with pytest.raises(ValueError):
        CA.prefix_attention(q, k[:1], v[:1], k, v, kv_lens=lens)
    with pytest.raises(ValueError):
        CA.cross_attention(q, k[0], v[0], cu_kv=torch.tensor([0.0, 2.5, 7.0]))
    kept = CA.cross_attention(q, k, v, kv_lens=[2, 3])
    for same in ((2, 3), torch.tensor([2, 3]), [torch.tensor(2), torch.tensor(3)], torch.tensor([2.0, 3.0]), range(2, 4)):
        assert torch.equal(CA.cross_attention(q, k, v, kv_lens=same), kept)


@gpu
@pytest.mark.parametrize("shape", [(2, 1, 8, 2, 128, 5000), (1, 300, 2, 2, 128, 3000), (30, 1, 8, 2, 64, 900)])
def test_split_calls_that_overlap_do_not_share_scratch(lib, shape):
    """Calls with a split key range and inputs of their own on two streams without an order between them, then two captured
    graphs replayed on the two: every result is that of the call alone."""
    B, Sq, H, Hkv, D, Skv = shape
    sides = []
    for seed in (21, 22):
        q, k, v = make(*shape, BF, "cuda", seed=seed)
        _, kp, vp = make(1, 1, 1, Hkv, D, 4000, BF, "cuda", seed=seed + 10)
        sides.append((q, k, v, kp, vp))

    def calls(q, k, v, kp, vp):
        return *CA.cross_attention(q, k, v, return_lse=True), *CA.prefix_attention(q, kp, vp, k, v, return_lse=True)

    alone = [calls(*s) for s in sides]
    assert not torch.equal(alone[0][0], alone[1][0])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(30):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(calls(*sides[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(a, b) for r in got[i] for a, b in zip(r, alone[i]))
    graphs, outs = [], []
    for s in sides:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(calls(*s))
    for _ in range(30):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(outs[i], alone[i]))


@gpu
def test_masks_too_long_for_the_bounded_waits_are_refused(lib):
    """One sample more than the limit; the largest masks below it are accepted, all hidden and all visible."""
    Skv, D = 1 << 23, 8
    kv = torch.zeros(17, Skv, 1, D, device="cuda", dtype=BF)
    q = torch.zeros(17, 40, 1, D, device="cuda", dtype=BF)
    for shown in (False, True):
        mask = torch.full((1, Skv), shown, device="cuda").expand(17, -1)
        with pytest.raises(native.NativeLibraryError):
            CA.cross_attention(q, kv, kv, key_mask=mask)
        o, lse = CA.cross_attention(q[:16], kv[:16], kv[:16], key_mask=mask[:16], return_lse=True)
        assert (o == 0).all() and ((lse - math.log(Skv)).abs() < 1e-4 if shown else lse == float("-inf")).all()
