"""Edges of the long-context operators on the GPU: values outside the ordinary
range, and waits that run out.  Plain 64-bit forms and tolerances as in longctx_ref.py."""
import ctypes as C
import decimal

import pytest
import torch

import longctx_ref as R
from inferno_b200._lib import InfernoError, call, lib

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _case(dtype, B, T, H, kv, d, P, lens, seed=0):
    """Sequences of lens[b] rows in slices of max(lens), weights gathered."""
    tid, dt = R.TYPES[dtype]
    g = _gen(seed)
    L = max(lens)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dt)

    c = dict(q=randn(B, T, H, d) * 2, out=torch.full((B, T, H, d), NAN, dtype=dt, device="cuda"))
    if P:
        c["pk"], c["pv"] = randn(P, kv, d), randn(P, kv, d)
    if L:
        c["k"], c["v"] = randn(B, L, kv, d), randn(B, L, kv, d)
        c["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        c["scores"] = torch.rand(B, kv, L, generator=g, device="cuda")
    return tid, c


def _run(tid, c):
    """Outputs of a call that leaves the case's own as they are."""
    c = dict(c, out=c["out"].clone())
    if "scores" in c:
        c["scores"] = c["scores"].clone()
    R.attention(R.attention_args(tid, **c))
    return c["out"], c.get("scores")


# ---------------------------------------------------------------------------
# weights do not depend on V
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,H,d,T", [("f32", 1, 256, 4), ("f32", 2, 128, 2), ("f32", 3, 64, 5), ("f32", 6, 256, 5),
                                         ("f32", 20, 128, 2), ("bf16", 2, 128, 3), ("f16", 8, 64, 4),
                                         ("bf16", 4, 256, 20), ("f32", 1, 256, 1), ("bf16", 2, 128, 1)])
@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("back", [0, 1])
def test_gathered_weights_do_not_depend_on_v(dtype, H, d, T, value, back):
    """An infinity or NaN in V of a row of the call's own tokens makes the outputs
    of the tokens that see it non-finite, and changes no weight and no other output."""
    if back >= T:
        pytest.skip("no such token")
    lens = [90, 33, T]
    tid, c = _case(dtype, 3, T, 2 * H, 2, d, 40, lens, seed=4)
    out, scores = _run(tid, c)
    for b, n in enumerate(lens):
        c["v"][b, n - 1 - back, 1, d // 3] = value
    got, got_scores = _run(tid, c)
    assert torch.equal(got_scores, scores) and scores.isfinite().all()
    blind = T - 1 - back
    assert torch.equal(got[:, :blind], out[:, :blind])
    assert torch.equal(got[:, :, :H], out[:, :, :H])                     # the other KV head
    assert not got[:, blind:, H:].isfinite().all(-1).any()


# ---------------------------------------------------------------------------
# infinite logits
# ---------------------------------------------------------------------------
INFINITE = [
    # type, batch, heads, kv, dim, prefix, lens
    ("f32", 1, 8, 2, 256, 0, [70]),                # CUDA cores, four rows
    ("f32", 3, 8, 2, 256, 300, [70, 1, 5]),        # eight and sixteen rows
    ("f32", 2, 4, 2, 128, 33, [9, 200]),
    ("f32", 1, 32, 2, 128, 0, [70]),               # tensor cores, one row tile
    ("f32", 2, 24, 1, 64, 200, [70, 64]),          # two, and four
    ("f32", 2, 17, 1, 256, 50, [33, 16]),
    ("bf16", 2, 8, 2, 128, 50, [70, 1]),
    ("f16", 2, 8, 2, 64, 50, [70, 33]),
    ("bf16", 24, 8, 2, 128, 3000, [1 + b for b in range(24)]),      # tcgen05
    ("f16", 24, 8, 2, 64, 6000, [40] * 24),
    ("bf16", 24, 8, 2, 256, 3000, [40] * 24),
]


@pytest.mark.parametrize("dtype,B,H,kv,d,P,lens", INFINITE)
def test_a_logit_of_minus_infinity_has_no_weight(dtype, B, H, kv, d, P, lens):
    """Whichever kernel takes the call: as if the row were not there."""
    tid, c = _case(dtype, B, 1, H, kv, d, P, lens, seed=7)
    c["q"][..., 0] = c["q"][..., 0].abs() + 0.5
    for b, n in enumerate(lens):
        c["k"][b, n - 1, :, 0] = -INF
    if P:
        c["pk"][0, :, 0] = -INF
    out, scores = _run(tid, c)
    less = [n - 1 for n in lens]
    want, tol, gathered, gtol = R.attention_ref(c["q"], less, c["k"], c["v"], c["pk"][1:] if P else None,
                                                c["pv"][1:] if P else None)
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"worst error / tolerance {float((err / tol).max())}"
    got = scores.double() - c["scores"].double()
    assert ((got - gathered).abs() <= gtol + scores.double() * 2.0 ** -24).all()
    for b, n in enumerate(lens):
        assert torch.equal(scores[b, :, n - 1:], c["scores"][b, :, n - 1:])


@pytest.mark.parametrize("dtype,B,H,kv,d,P,lens", INFINITE)
def test_logits_of_minus_infinity_alone_give_zeros(dtype, B, H, kv, d, P, lens):
    tid, c = _case(dtype, B, 1, H, kv, d, P, lens, seed=6)
    c["q"][..., 0] = c["q"][..., 0].abs() + 0.5
    c["k"][..., 0] = -INF
    if P:
        c["pk"][..., 0] = -INF
    out, scores = _run(tid, c)
    assert (out == 0).all() and torch.equal(scores, c["scores"])


@pytest.mark.parametrize("dtype,B,H,kv,d,P,lens", INFINITE)
def test_a_logit_of_infinity_spoils_its_row(dtype, B, H, kv, d, P, lens):
    """NaN for the heads that see it, the same bits for the others."""
    tid, c = _case(dtype, B, 1, H, kv, d, P, lens, seed=8)
    c["q"][..., 0] = c["q"][..., 0].abs() + 0.5
    out, scores = _run(tid, c)
    c["k"][0, lens[0] // 2, 0, 0] = INF
    got, got_scores = _run(tid, c)
    G = H // kv
    assert got[0, 0, :G].isnan().all() and got_scores[0, 0, :lens[0]].isnan().all()
    assert torch.equal(got[1:], out[1:]) and torch.equal(got[0, 0, G:], out[0, 0, G:])
    assert torch.equal(got_scores[1:], scores[1:]) and torch.equal(got_scores[0, 1:], scores[0, 1:])


# ---------------------------------------------------------------------------
# weights far below the largest
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("weight", [4.5e-8, 1e-7, 1e-6, 1e-4])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("B,H,d,P,lens", [
    (1, 4, 64, 0, [777]), (1, 20, 128, 0, [333]), (1, 40, 256, 0, [100]),      # one, two and four row tiles of own rows
    (2, 4, 128, 1000, [1, 1]),                                                 # a prefix of few query rows
    (16, 4, 64, 16001, [1] * 16), (16, 4, 128, 4097, [1] * 16), (16, 4, 256, 3001, [1] * 16),      # and of many
])
def test_attention_small_weights_add_up(dtype, weight, B, H, d, P, lens):
    """Every 16th key takes nearly all the weight and holds V = 0: what is left is
    the sum over keys of a small weight each.  (P in fp16 keeps its half step down
    to 2^-14 of what it is scaled to: 2^-25 of the largest at least.)"""
    tid, c = _case(dtype, B, 1, H, 1, d, P, lens, seed=9)
    c["q"].zero_()
    c["q"][..., 0] = 4.0
    high = torch.log(torch.tensor(1 / weight)).item() / 4.0
    for k, v in ((c["k"], c["v"]), (c.get("pk"), c.get("pv"))):
        if k is None:
            continue
        k.zero_()
        v.copy_((torch.rand(v.shape, generator=_gen(3), device="cuda") + 1) * 16384)
        rows = k.dim() - 3                           # [rows][kv][dim] or [batch][rows][kv][dim]
        if k.shape[rows] > 1:
            (k if rows == 0 else k.transpose(0, 1))[::16, ..., 0] = high
            (v if rows == 0 else v.transpose(0, 1))[::16] = 0
        else:
            v.zero_()
    c.pop("scores")
    R.attention(R.attention_args(tid, scale=1.0, **c))
    want, tol, _, _ = R.attention_ref(c["q"], lens, c["k"], c["v"], c.get("pk"), c.get("pv"), 1.0)
    assert (want > 100 * torch.finfo(c["out"].dtype).smallest_normal).all()
    err = (c["out"].double() - want).abs()
    assert (err <= tol).all(), f"worst error / tolerance {float((err / tol).max())}"


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("B,H,d,P,lens", [
    (1, 4, 64, 0, [777]), (1, 20, 128, 0, [333]), (1, 40, 256, 0, [100]), (2, 4, 128, 1000, [1, 1]),
    (16, 4, 64, 16001, [1] * 16), (16, 4, 128, 4097, [1] * 16), (16, 4, 256, 3001, [1] * 16)])
def test_attention_huge_logits(dtype, B, H, d, P, lens):
    """Logits of up to 1e8 (and, scaled, 1e10), whose steps in fp32 are 8 and more: the
    largest takes all the weight, the others being thousands below, and the output is
    its V: bit for bit in 16 bits, in fp32 to the 2^-19 that the pair products keep."""
    tid, c = _case(dtype, B, 1, H, 1, d, P, lens, seed=10)
    for n in ("q", "k", "pk"):
        if n in c:
            c[n].copy_(torch.randint(-7, 8, c[n].shape, generator=_gen(len(n)), device="cuda") * 1000.0)
    c.pop("scores")
    for scale in (d ** -0.5, -100.0):
        R.attention(R.attention_args(tid, scale=scale, **c))
        for b, n in enumerate(lens):
            keys = torch.cat([c["pk"][:, 0], c["k"][b, :n, 0]] if P else [c["k"][b, :n, 0]]).double()
            vals = torch.cat([c["pv"][:, 0], c["v"][b, :n, 0]] if P else [c["v"][b, :n, 0]])
            top = (c["q"][b, 0].double() @ keys.t() * scale).topk(2, -1)
            sure = top.values[:, 0] - top.values[:, 1] > 1e4
            assert sure.any()
            got, want = c["out"][b, 0][sure], vals[top.indices[:, 0]][sure]
            assert torch.equal(got, want) if dtype != "f32" else ((got - want).abs() <= want.abs() * 2.0 ** -19).all()


# ---------------------------------------------------------------------------
# far positions
# ---------------------------------------------------------------------------
def _far_angles(positions, rope_dim, theta, factors=None):
    """Angles within [-pi, pi] from 60 decimal digits."""
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        two_pi = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
        log = decimal.Decimal(theta).ln()
        rows = []
        for at in positions:
            row = []
            for i in range(rope_dim // 2):
                a = at * (-log * 2 * i / rope_dim).exp()
                if factors is not None:
                    a /= decimal.Decimal(factors[i])
                row.append(float(a - (a / two_pi).to_integral_value() * two_pi))
            rows.append(row)
    return torch.tensor(rows, dtype=torch.float64)


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("theta,r,with_factors", [(1e4, 512, False), (1.5, 512, False), (2.0, 64, True), (5e5, 128, True)])
def test_rope_far_positions(theta, r, with_factors, layout):
    """fp32 up to position 2^31 - 1.  The turn is exact to 2^-26 from its rounding
    to fp32 and 2^-26 from the frequency (2^-54 of itself, 2^28.4 turns at most): 2 pi
    2^-25 in the angle, which moves a value by at most |a| + |b| of it; sincospi is
    off by 2 ulp (2^-23); two products and a sum round (3 * 2^-24)."""
    n, H = 3, 2
    positions = [(1 << 31) - 1, 1234567891, 3]
    g = _gen(11)
    x = torch.randn(n, H * r, generator=g, device="cuda")
    pos = torch.tensor(positions, dtype=torch.int32, device="cuda")
    ff = torch.rand(r // 2, generator=g, device="cuda") + 0.75 if with_factors else None
    y = torch.empty_like(x)
    R.rope(R.rope_args(0, x, None, None, y, n_tokens=n, n_heads=H, n_kv_heads=0, head_dim=r, rope_dim=r, positions=pos,
                       layout=layout, theta=theta, freq_factors=R.ptr(ff)))
    ang = _far_angles(positions, r, theta, ff.tolist() if with_factors else None)
    want, mass = R.rope_ref(x.view(n, H, r), ang, 1.0, r, layout)
    tol = mass * (6.2832 * 2.0 ** -25 + 2.0 ** -23 + 3 * 2.0 ** -24)
    err = (y.view(n, H, r).double().cpu() - want).abs()
    assert (err <= tol).all(), f"worst error / tolerance {float((err / tol).max())}"


@pytest.mark.parametrize("layout", [0, 1])
def test_rope_infinite_factor_and_negative_positions(layout):
    """A pair whose factor is infinite does not turn; a negative position turns back,
    with factors and without (the same angle, so the same bits)."""
    n, r = 4, 32
    g = _gen(13)
    x = torch.randn(n, r, generator=g, device="cuda")
    pos = torch.tensor([1, 77, 123456, 1 << 30], dtype=torch.int32, device="cuda")
    ff = torch.full((r // 2,), INF, device="cuda")
    kw = dict(n_tokens=n, n_heads=1, n_kv_heads=0, head_dim=r, rope_dim=r, theta=1e4, layout=layout)
    y, z = torch.empty_like(x), torch.empty_like(x)
    R.rope(R.rope_args(0, x, None, None, y, positions=pos, freq_factors=R.ptr(ff), **kw))
    assert torch.equal(y, x)
    for f in (None, torch.full_like(ff, 1.25)):
        R.rope(R.rope_args(0, x, None, None, y, positions=pos, inverse=1, freq_factors=R.ptr(f), **kw))
        R.rope(R.rope_args(0, x, None, None, z, positions=-pos, freq_factors=R.ptr(f), **kw))
        assert torch.equal(y, z)


@pytest.mark.parametrize("with_factors", [False, True])
@pytest.mark.parametrize("theta", [1.1, 1e4])
def test_rope_more_than_a_turn_per_position(theta, with_factors):
    """A factor below 1 / (2 pi) gives pairs of more than one turn per position.  20
    turns times 5000 positions are exact to 2^-36 in either form, so the tolerance is
    that of the fp32 steps: 2 pi 2^-26 in the angle, 2^-23, 3 * 2^-24; the plain form's
    angles of up to 7e5 are off by 2^-33."""
    n, r = 6, 64
    g = _gen(14)
    x = torch.randn(n, r, generator=g, device="cuda")
    pos = torch.tensor([0, 1, 2, 999, 4321, 5000], dtype=torch.int32, device="cuda")
    ff = torch.rand(r // 2, generator=g, device="cuda") + 0.5 if with_factors else None
    y = torch.empty_like(x)
    R.rope(R.rope_args(0, x, None, None, y, n_tokens=n, n_heads=1, n_kv_heads=0, head_dim=r, rope_dim=r, positions=pos,
                       theta=theta, scaling=1, factor=0.0078125, freq_factors=R.ptr(ff)))
    theta = float(torch.tensor(theta))                         # as the struct holds it
    ang, _ = R.rope_angles(pos, r, theta, scaling=1, factor=0.0078125, freq_factors=ff)
    want, mass = R.rope_ref(x.view(n, 1, r), ang, 1.0, r, 0)
    err = (y.view(n, 1, r).double().cpu() - want).abs()
    assert (err <= mass * (6.2832 * 2.0 ** -26 + 2.0 ** -23 + 3 * 2.0 ** -24 + 2.0 ** -30)).all()


@pytest.mark.parametrize("with_factors", [False, True])
@pytest.mark.parametrize("factor,orig_ctx", [(0.125, 8), (0.0078125, 30), (0.5, 4096)])
def test_rope_by_parts_with_a_factor_below_one(factor, orig_ctx, with_factors):
    """Later pairs then turn faster than the first.  Tolerance as above, with 7e5 of
    angle at most."""
    n, r = 6, 64
    g = _gen(15)
    x = torch.randn(n, r, generator=g, device="cuda")
    pos = torch.tensor([0, 1, 2, 999, 4321, 5000], dtype=torch.int32, device="cuda")
    ff = torch.rand(r // 2, generator=g, device="cuda") + 0.5 if with_factors else None
    y = torch.empty_like(x)
    kw = dict(scaling=2, factor=factor, orig_ctx=orig_ctx)
    R.rope(R.rope_args(0, x, None, None, y, n_tokens=n, n_heads=1, n_kv_heads=0, head_dim=r, rope_dim=r, positions=pos,
                       theta=1e4, freq_factors=R.ptr(ff), **kw))
    ang, gain = R.rope_angles(pos, r, 1e4, freq_factors=ff, **kw)
    want, mass = R.rope_ref(x.view(n, 1, r), ang, gain, r, 0)
    err = (y.view(n, 1, r).double().cpu() - want).abs()
    assert (err <= mass * (6.2832 * 2.0 ** -26 + 2.0 ** -23 + 3 * 2.0 ** -24 + 2.0 ** -30)).all()


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("scale", [dict(scaling=2, factor=8.0, orig_ctx=4096), dict(mscale=1.5)])
def test_rope_inverse_with_a_gain(scale, layout):
    """The inverse carries the forward call's factor m of cos and sin: it is the
    gradient.  With mscale 1 / m it undoes the forward call."""
    n, H, d, r = 5, 2, 64, 32
    g = _gen(2)
    w, x = torch.randn(n, H * d, generator=g, device="cuda"), torch.randn(n, H * d, generator=g, device="cuda")
    pos = torch.tensor([0, 5, 90000, 77, 4095], dtype=torch.int32, device="cuda")
    kw = dict(n_tokens=n, n_heads=H, n_kv_heads=0, head_dim=d, rope_dim=r, positions=pos, theta=1e4, layout=layout, **scale)
    ang, m = R.rope_angles(pos, r, 1e4, **scale)
    assert m != 1.0
    # sincospi, the angle, m's own rounding and the products: 2^-21 of the pair's mass (see test_longctx_gpu.py)
    got = torch.empty_like(w)
    R.rope(R.rope_args(0, w, None, None, got, inverse=1, **kw))
    want = torch.zeros(n, H, d, dtype=torch.float64)
    wd = w.double().cpu().view(n, H, d)
    for i in range(d):
        unit = torch.zeros(n, H, d, dtype=torch.float64)
        unit[..., i] = 1.0
        up, down = R.rope_ref(unit, ang, m, r, layout)[0], R.rope_ref(-unit, ang, m, r, layout)[0]
        want[..., i] = ((up - down) / 2 * wd).sum(-1)
    _, mass = R.rope_ref(wd, ang, m, r, layout)
    assert ((got.double().cpu().view(n, H, d) - want).abs() <= mass * 2.0 ** -21 + want.abs() * 2.0 ** -23).all()
    y, z = torch.empty_like(x), torch.empty_like(x)
    R.rope(R.rope_args(0, x, None, None, y, **kw))
    R.rope(R.rope_args(0, y, None, None, z, inverse=1, **{**kw, "mscale": 1 / m}))
    _, mass = R.rope_ref(x.view(n, H, d), ang, 1.0, r, layout)
    # two rotations, the second of values of up to mass, and m 1 / m rounded
    assert ((z - x).view(n, H, d).double().cpu().abs() <= mass * 2.0 ** -19 + 1e-30).all()


# ---------------------------------------------------------------------------
# buffers that the device cannot read
# ---------------------------------------------------------------------------
def _calls():
    """Valid calls of the three operators and what keeps their buffers alive."""
    B, H, kv, d, L = 2, 4, 2, 64, 40
    dev = dict(device="cuda")
    x = {n: torch.zeros(B, 1, h, d, dtype=torch.bfloat16, **dev) for n, h in (("q", H), ("out", H), ("k", kv), ("v", kv))}
    x.update({n: torch.zeros(B, L, kv, d, dtype=torch.bfloat16, **dev) for n in ("kc", "vc")})
    x.update({n: torch.zeros(20, kv, d, dtype=torch.bfloat16, **dev) for n in ("pk", "pv")})
    x.update({n: torch.zeros(B, kv, L, **dev) for n in ("scores", "scores_out")})
    x.update({n: torch.zeros(B, kv, L, dtype=torch.int32, **dev) for n in ("pos", "pos_out")})
    x.update({n: torch.full((B,), 30, dtype=torch.int32, **dev) for n in ("lens", "next_pos", "lens_out", "slots")})
    x["slots"][1] = 70
    x["ff"] = torch.ones(d // 2, **dev)
    rope = R.rope_args(30, x["q"].view(B, -1), x["k"].view(B, -1), x["v"].view(B, -1), x["out"].view(B, -1),
                       x["kc"].view(B * L, -1), x["vc"].view(B * L, -1), n_tokens=B, n_heads=H, n_kv_heads=kv, head_dim=d,
                       rope_dim=d, positions=x["lens"], theta=1e4, slots=R.ptr(x["slots"]), n_rows=B * L,
                       freq_factors=R.ptr(x["ff"]))
    attn = R.attention_args(30, x["q"], x["out"], x["lens"], x["kc"], x["vc"], x["pk"], x["pv"], x["scores"])
    evict = R.evict_args(30, x["kc"], x["vc"], x["scores"], x["pos"], x["lens"], x["next_pos"], x["scores_out"],
                         x["pos_out"], x["lens_out"], budget=16)
    x["ws"] = torch.empty(max(R.attention_workspace(attn).numel(), R.evict_workspace(evict).numel()), dtype=torch.uint8, **dev)
    ws, n = C.c_void_p(x["ws"].data_ptr()), x["ws"].numel()
    return x, {"inferno_rope": (rope, lambda a: ()), "inferno_attention_cached": (attn, lambda a: (ws, n)),
               "inferno_cache_evict": (evict, lambda a: (ws, n))}


@pytest.mark.parametrize("fn,fields", [
    ("inferno_rope", "q k v q_out k_out v_out positions slots freq_factors"),
    ("inferno_attention_cached", "q out prefix_k prefix_v k_cache v_cache lens scores"),
    ("inferno_cache_evict", "k_cache v_cache scores slot_pos lens next_pos scores_out slot_pos_out lens_out")])
def test_any_buffer_in_host_memory_is_refused(fn, fields):
    _, calls = _calls()
    a, more = calls[fn]
    host = torch.zeros(1 << 16)
    call(fn, C.byref(a), *more(a), R.stream())
    for field in fields.split():
        good = getattr(a, field)
        setattr(a, field, host.data_ptr())
        with pytest.raises(InfernoError, match="not device memory"):
            call(fn, C.byref(a), *more(a), R.stream())
        setattr(a, field, good)
    if fn != "inferno_rope":
        size = getattr(lib(), fn + "_workspace")(C.byref(a))
        store = torch.zeros(size + 256, dtype=torch.uint8)
        at = (store.data_ptr() + 255) // 256 * 256
        with pytest.raises(InfernoError, match="not device memory"):
            call(fn, C.byref(a), C.c_void_p(at), size, R.stream())
    call(fn, C.byref(a), *more(a), R.stream())


def test_pinned_lengths_are_read():
    """Pinned host memory is memory of CUDA's, which a kernel can read."""
    tid, c = _case("bf16", 3, 1, 4, 2, 64, 40, [90, 33, 1], seed=2)
    out, scores = _run(tid, c)
    got, got_scores = _run(tid, dict(c, lens=c["lens"].cpu().pin_memory()))
    torch.cuda.synchronize()
    assert torch.equal(got, out) and torch.equal(got_scores, scores)


# ---------------------------------------------------------------------------
# what the next position protects
# ---------------------------------------------------------------------------
def test_evict_protects_the_recent_rows_before_the_next_position():
    """A decode step that advances its positions before it evicts keeps its first
    n_sink and last n_recent rows, and no other where the budget has no more; with the
    positions of the tokens just appended one row more is protected, and the rows of
    both kinds, now more than the budget, compete by weight."""
    B, kv, L, sink, recent = 2, 2, 60, 3, 9
    k, v = (torch.zeros(B, L, kv, 64, device="cuda") for _ in range(2))
    scores = torch.arange(L, 0, -1, device="cuda").float().expand(B, kv, L).contiguous()      # the newest weigh least
    pos = torch.arange(L, device="cuda", dtype=torch.int32).expand(B, kv, L).contiguous()
    for ahead, kept in ((0, list(range(sink)) + list(range(L - recent, L))),
                        (-1, list(range(sink)) + list(range(L - recent - 1, L - 1)))):
        lens = torch.full((B,), L, dtype=torch.int32, device="cuda")
        nxt = torch.full((B,), L + ahead, dtype=torch.int32, device="cuda")
        so, po, lo = torch.zeros_like(scores), torch.zeros_like(pos), torch.zeros_like(lens)
        R.evict(R.evict_args(0, k, v, scores, pos, lens, nxt, so, po, lo, budget=sink + recent, n_sink=sink, n_recent=recent))
        for b in range(B):
            for h in range(kv):
                assert sorted(po[b, h, :sink + recent].tolist()) == kept


# ---------------------------------------------------------------------------
# waits that run out
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,B,H,kv,d,P", [("bf16", 24, 8, 2, 128, 3000), ("f16", 24, 8, 2, 64, 6000),
                                              ("bf16", 40, 8, 2, 256, 3000)])
def test_a_wait_that_runs_out_gives_nan(dtype, B, H, kv, d, P):
    """Whatever an earlier call left in the workspace: NaN outputs and weights, the
    device error word set, and the next call as ever."""
    tid, c = _case(dtype, B, 1, H, kv, d, P, [40] * B, seed=5)
    a = R.attention_args(tid, **c)
    ws = R.attention_workspace(a)
    before = c["scores"].clone()
    R.attention(a, ws)
    want, want_scores = c["out"].clone(), c["scores"].clone()
    c["scores"].copy_(before)
    assert lib().inferno_device_error(0, 1) == 0
    call("inferno_debug_attention_timeout", C.byref(a), C.c_void_p(ws.data_ptr()), ws.numel(), R.stream())
    assert c["out"].isnan().all() and c["scores"].isnan().all()
    assert lib().inferno_device_error(0, 1) == 1
    c["scores"].copy_(before)
    R.attention(a, ws)
    assert torch.equal(c["out"], want) and torch.equal(c["scores"], want_scores)
    assert lib().inferno_device_error(0, 0) == 0
