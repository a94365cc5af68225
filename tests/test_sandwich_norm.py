"""`rmsnorm_gate_residual_modulate` against the two-step chain and the definition in 64 bits."""
import pytest
import torch

from telefuser_b200.ops import functional as TF
from telefuser_b200.ops import native

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def inputs(B, S, C, dtype, device, tables="sample", seed=0, wtype=None):
    g = torch.Generator(device=device).manual_seed(seed)
    n = {"sample": (B, 1), "token": (B, S), "one": (1, 1)}[tables]
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    wtype = wtype or dtype
    return dict(res=(2 * r(B, S, C)).to(dtype), y=r(B, S, C).to(dtype), weight=(1 + 0.1 * r(C)).to(wtype), gate=0.7 * r(*n, C),
                next_weight=(1 + 0.1 * r(C)).to(wtype), shift=0.3 * r(*n, C), scale=0.3 * r(*n, C))  # fmt: skip


def check(x, h, a, eps=1e-6, tanh_gate=True, post_norm=True):
    """x within half a step of the type and fp32's own error (a sum of up to 8192 squares in pairs, rsqrt, tanh and five
    products: 2^-19 of the terms); h the same from x as it was stored."""
    d = {k: None if t is None else t.double() for k, t in a.items()}
    u = torch.finfo(a["res"].dtype).eps / 2
    n = d["y"]
    if post_norm:
        n = n * torch.rsqrt(n.square().mean(-1, keepdim=True) + eps) * (1 if d["weight"] is None else d["weight"])
    if d["gate"] is not None:
        n = n * (d["gate"].tanh() if tanh_gate else d["gate"])
    want = d["res"] + n
    assert ((x.double() - want).abs() <= u * want.abs() + 2.0**-19 * (d["res"].abs() + n.abs()) + torch.finfo(x.dtype).tiny).all()
    xd = x.double()
    hw = xd * torch.rsqrt(xd.square().mean(-1, keepdim=True) + eps) * (1 if d["next_weight"] is None else d["next_weight"])
    hs = hw if d["scale"] is None else hw * (1 + d["scale"])
    want = hs if d["shift"] is None else hs + d["shift"]
    size = hw.abs() * (1 if d["scale"] is None else 1 + d["scale"].abs()) + (0 if d["shift"] is None else d["shift"].abs())
    assert ((h.double() - want).abs() <= u * want.abs() + 2.0**-19 * size + torch.finfo(h.dtype).tiny).all()


# ---- CPU --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tanh", [True, False])
def test_equals_the_two_step_chain_on_cpu(tanh):
    a = inputs(2, 5, 24, torch.bfloat16, "cpu")
    x, h = TF.rmsnorm_gate_residual_modulate(**a, tanh_gate=tanh)
    x2 = TF.rmsnorm_gate_residual(a["res"], a["y"], a["weight"], a["gate"], tanh_gate=tanh)
    assert torch.equal(x, x2)
    assert torch.equal(h, TF.rmsnorm_modulate(x2, a["next_weight"], a["shift"], a["scale"]))


def test_without_the_first_norm_on_cpu():
    a = inputs(2, 5, 24, torch.bfloat16, "cpu", "token")
    a["weight"] = None
    x, h = TF.rmsnorm_gate_residual_modulate(**a, tanh_gate=False, post_norm=False)
    x2 = TF.gated_residual(a["res"], a["y"], a["gate"])
    assert torch.equal(x, x2)
    assert torch.equal(h, TF.rmsnorm_modulate(x2, a["next_weight"], a["shift"], a["scale"]))


@pytest.mark.parametrize("change", [
    dict(y=torch.zeros(2, 5, 16)), dict(y=torch.zeros(2, 5, 24, dtype=torch.float64)), dict(weight=torch.ones(23)),
    dict(next_weight=torch.ones(1, 24)), dict(post_norm=False),
])  # fmt: skip
def test_refusals(change):
    a = inputs(2, 5, 24, torch.float32, "cpu") | change
    with pytest.raises(ValueError):
        TF.rmsnorm_gate_residual_modulate(**a)


@pytest.mark.parametrize("shape", [(1, 5, 24), (1, 2, 24), (2, 24), (5, 24), (5, 1, 24), (2, 2, 24), (2, 1, 16), (48,)])
@pytest.mark.parametrize("which", ["gate", "shift", "scale"])
@pytest.mark.parametrize("S", [5, 2])
def test_tables_that_repeat_in_no_documented_way_are_refused(shape, which, S):
    a = inputs(2, S, 24, torch.float32, "cpu")
    if shape == (2, S, 24):
        return
    with pytest.raises(ValueError):
        TF.rmsnorm_gate_residual_modulate(**(a | {which: torch.zeros(shape)}))


@pytest.mark.parametrize("shape", [(24,), (1, 24), (1, 1, 24), (2, 1, 24), (2, 2, 24)])
def test_tables_that_fit(shape):
    a = inputs(2, 2, 24, torch.float32, "cpu") | dict(scale=torch.randn(shape))
    check(*TF.rmsnorm_gate_residual_modulate(**a), a)


# ---- GPU --------------------------------------------------------------------------------------------------------------
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tables", ["sample", "token", "one"])
@pytest.mark.parametrize("B,S,C", [(1, 1, 8), (1, 3, 2048), (2, 77, 3840), (3, 5, 40), (2, 1001, 264), (1, 300, 4104), (2, 9, 8192), (2, 700, 3840), (3, 500, 72), (1, 1300, 5120), (40, 33, 2048)])
def test_matches_the_definition(B, S, C, tables, dtype):
    a = inputs(B, S, C, dtype, "cuda", tables)
    check(*TF.rmsnorm_gate_residual_modulate(**a), a)
    check(*TF.rmsnorm_gate_residual_modulate(**a, tanh_gate=False, eps=1e-3), a, tanh_gate=False, eps=1e-3)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("absent", [(), ("gate",), ("shift",), ("scale",), ("weight", "next_weight"), ("gate", "shift", "scale")])
@pytest.mark.parametrize("post", [True, False])
def test_optional_parts(absent, post, dtype):
    a = inputs(2, 700, 520, dtype, "cuda") | {k: None for k in absent}
    if not post:
        a["weight"] = None
    check(*TF.rmsnorm_gate_residual_modulate(**a, post_norm=post), a, post_norm=post)


@gpu
def test_strided_inputs_weights_of_another_type_and_table_slices():
    a = inputs(2, 40, 128, torch.bfloat16, "cuda", wtype=torch.float32)
    wide = torch.cat([a["res"], a["y"]], dim=-1)
    tab = torch.cat([a["gate"], a["shift"], a["scale"]], dim=-1)  # [B, 1, 3 C], the block's modulation
    b = a | dict(res=wide[..., :128], y=wide[..., 128:], gate=tab[..., :128], shift=tab[..., 128:256], scale=tab[..., 256:])
    check(*TF.rmsnorm_gate_residual_modulate(**b), a)
    b["next_weight"] = a["next_weight"].bfloat16()
    check(*TF.rmsnorm_gate_residual_modulate(**b), a | dict(next_weight=b["next_weight"]))
    odd = torch.empty(a["y"].numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view(a["y"].shape).copy_(a["y"])
    check(*TF.rmsnorm_gate_residual_modulate(**(a | dict(y=odd, res=a["res"].transpose(0, 1).contiguous().transpose(0, 1)))), a)
    mixed = a | dict(gate=a["gate"][:1], shift=inputs(2, 40, 128, torch.bfloat16, "cuda", "token")["shift"])
    check(*TF.rmsnorm_gate_residual_modulate(**mixed), mixed)
    with pytest.raises(ValueError):
        TF.rmsnorm_gate_residual_modulate(**(a | dict(gate=torch.zeros(3, 1, 128, device="cuda"))))


@gpu
def test_odd_widths_take_the_reference_steps_and_empty_inputs_return():
    a = inputs(2, 3, 20, torch.bfloat16, "cuda")
    check(*TF.rmsnorm_gate_residual_modulate(**a), a)
    x, h = TF.rmsnorm_gate_residual_modulate(torch.empty(2, 0, 64, device="cuda"), torch.empty(2, 0, 64, device="cuda"))
    assert x.shape == h.shape == (2, 0, 64)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_zero_rows_and_large_values(dtype):
    a = inputs(1, 6, 1024, dtype, "cuda")
    a["y"][0, 1] = 0
    a["res"][0, 2] = 0
    a["y"][0, 2] = 0
    a["res"][0, 3] *= 1e4
    a["y"][0, 4] *= 1e4
    check(*TF.rmsnorm_gate_residual_modulate(**a), a)


@gpu
def test_same_bits_again_and_replayed():
    a = inputs(2, 500, 2048, torch.bfloat16, "cuda")
    x, h = TF.rmsnorm_gate_residual_modulate(**a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        xg, hg = TF.rmsnorm_gate_residual_modulate(**a)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, xg) and torch.equal(h, hg)
    assert native.last_status() == 0


# ---- expanded tables --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("base,shape,rows_per", [
    ((1, 1, 32), (1, 37, 32), 37), ((1, 1, 32), (3, 37, 32), 111), ((3, 1, 32), (3, 37, 32), 37), ((32,), (3, 37, 32), 111),
    ((1, 1, 32), (3, 1, 32), 111), ((3, 37, 32), (3, 37, 32), 1), ((1, 37, 32), (3, 37, 32), 1), ((1, 37, 32), (1, 37, 32), 1),
    ((1, 1, 1), (3, 37, 32), 111), ((3, 37, 1), (3, 37, 32), 1),
])  # fmt: skip
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_an_expanded_table_repeats_are_taken_once(base, shape, rows_per, dtype):
    acts = torch.empty(3, 37, 32) if shape[0] == 3 else torch.empty(1, 37, 32)
    rows = acts.numel() // 32
    wide = torch.randn(*base[:-1], 2 * base[-1] if base[-1] > 1 else 1).to(dtype)
    view = wide[..., : base[-1]].expand(shape)  # a slice of a wider table, expanded
    t, at, ld, per = TF._row_table(view, acts.shape, rows, 32)
    assert per == rows_per and ld % 4 == 0 and at % 16 == 0 and at == t.data_ptr()
    flat = torch.as_strided(t, (rows // per, 32), (ld, 1))
    assert torch.equal(flat.repeat_interleave(per, dim=0), view.float().expand(acts.shape).reshape(rows, 32))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_expanded_tables(dtype):
    a = inputs(3, 500, 264, dtype, "cuda")
    small = {k: a[k].clone() for k in ("gate", "shift", "scale")}
    a["gate"], a["shift"] = small["gate"].expand(3, 500, 264), small["shift"][:1].expand(3, 500, 264)
    a["scale"] = small["scale"][:1].expand(3, 1, 264)
    x, h = TF.rmsnorm_gate_residual_modulate(**a)
    check(x, h, a)
    b = a | dict(gate=small["gate"], shift=small["shift"][:1], scale=small["scale"][:1])
    assert all(torch.equal(s, t) for s, t in zip((x, h), TF.rmsnorm_gate_residual_modulate(**b)))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,S,C", [(1200, 1, 264), (600, 2, 2048), (700, 3, 1024), (301, 4, 3840), (211, 7, 520), (211, 8, 520), (300, 4, 5120), (600, 2, 4104), (75, 17, 1024)])
def test_many_samples_of_few_rows(B, S, C, dtype):
    a = inputs(B, S, C, dtype, "cuda")
    check(*TF.rmsnorm_gate_residual_modulate(**a), a)
    one = a | dict(gate=a["gate"][:1].expand(B, S, C), shift=a["shift"][:1], scale=a["scale"].expand(B, S, C))
    check(*TF.rmsnorm_gate_residual_modulate(**one), one)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("shape", [(24,), (5, 24), (2, 5, 24)])
@pytest.mark.parametrize("extra", [0, 1, 3])
def test_one_row_for_all_keeps_the_shape_of_the_activations(shape, extra, device):
    g = torch.Generator().manual_seed(0)
    a = {n: torch.randn(*shape, generator=g).to(device) for n in ("res", "y")}
    a |= {n: torch.randn(*(1,) * extra, 24, generator=g).to(device) for n in ("gate", "shift", "scale")} | dict(weight=None, next_weight=None)
    x, h = TF.rmsnorm_gate_residual_modulate(**a)
    assert x.shape == h.shape == shape
    check(x, h, {k: v.reshape(24) if k in ("gate", "shift", "scale") else v for k, v in a.items()})


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("shape,table", [((0, 5, 24), (0, 1, 24)), ((0, 5, 24), (1, 1, 24)), ((2, 0, 24), (2, 1, 24)), ((2, 0, 24), (2, 0, 24))])
def test_empty_activations_with_tables(shape, table, device):
    z = torch.zeros(shape, device=device)
    x, h = TF.rmsnorm_gate_residual_modulate(z, z, gate=torch.zeros(table, device=device), scale=torch.zeros(24, device=device))
    assert x.shape == h.shape == shape
