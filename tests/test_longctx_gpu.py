"""GPU parity of the long-context operators with their plain 64-bit forms
(longctx_ref.py), through the C ABI, at the sizes and masks where they can go
wrong; tolerances count roundings (see attention_ref)."""
import ctypes as C

import pytest
import torch

import longctx_ref as R
from inferno_b200._lib import InfernoError, call, lib

pytestmark = pytest.mark.gpu
NAN = float("nan")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, dt, *shape):
    return torch.randn(*shape, generator=g, device="cuda").to(dt)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def _rope_tol(mass, want, dt):
    """The turn's fraction rounds to 2^-26, 2 pi 2^-26 < 2^-23 in the angle;
    sincospi is off by 2 ulp at most (2^-22 of values up to 1); the products and
    their sum round three times and gain once (2^-24 each): 2^-21 (|a| + |b|) in
    all.  The output rounds once."""
    return mass * 2.0 ** -21 + want.abs() * R.half_step(dt) + torch.finfo(dt).smallest_normal


ROPE = [
    # type, tokens, heads, kv, dim, rope_dim, interleaved, positions up to, scaling
    ("f32", 1, 8, 2, 256, 64, 0, 1000, {}),
    ("f32", 5, 3, 1, 20, 10, 0, 1 << 20, {}),                      # rows of 80 bytes, halves of 20
    ("f32", 7, 1, 1, 33, 2, 1, 4096, {}),                          # odd head_dim
    ("f32", 1000, 4, 4, 96, 96, 1, 100000, dict(scaling=1, factor=4.0)),
    ("bf16", 1, 32, 8, 128, 128, 0, (1 << 31) - 1, {}),
    ("bf16", 777, 28, 4, 128, 128, 1, 131072, dict(scaling=2, factor=8.0)),
    ("bf16", 64, 6, 2, 80, 20, 0, 9000, {}),
    ("f16", 300, 16, 2, 64, 64, 0, 32768, dict(scaling=2, factor=4.0, orig_ctx=2048, beta_fast=16.0, beta_slow=2.0)),
    ("f16", 33, 5, 5, 512, 512, 1, 70000, dict(scaling=2, factor=0.5)),
    ("f16", 2, 2, 1, 10, 6, 1, 77, dict(mscale=1.5)),
    ("f32", 3, 0, 4, 64, 32, 0, 5000, {}),                         # k alone
    ("bf16", 3, 4, 0, 64, 64, 0, 5000, {}),                        # q alone
]


@pytest.mark.parametrize("dtype,n,H,kv,d,r,ilv,far,scale", ROPE)
def test_rope(dtype, n, H, kv, d, r, ilv, far, scale):
    tid, dt = R.TYPES[dtype]
    g = _gen(n + d)
    q, k = _randn(g, dt, n, max(H, 1) * d), _randn(g, dt, n, max(kv, 1) * d)
    pos = torch.randint(0, far, (n,), generator=g, device="cuda", dtype=torch.int32)
    pos[0] = far - 1
    qo, ko = torch.full_like(q, NAN), torch.full_like(k, NAN)
    theta = 1e7 if d == 256 else 1e4
    R.rope(R.rope_args(tid, q if H else None, k if kv else None, None, qo if H else None, ko if kv else None,
                       n_tokens=n, n_heads=H, n_kv_heads=kv, head_dim=d, rope_dim=r, positions=pos, layout=ilv,
                       theta=theta, **{"orig_ctx": 4096, **scale}))
    ang, gain = R.rope_angles(pos, r, theta, **scale)
    for heads, x, y in ((H, q, qo), (kv, k, ko)):
        if not heads:
            assert y.isnan().all()
            continue
        want, mass = R.rope_ref(x.view(n, heads, d), ang, gain, r, ilv)
        err = (y.view(n, heads, d).double().cpu() - want).abs()
        assert (err <= _rope_tol(mass, want, dt)).all(), float((err - _rope_tol(mass, want, dt)).max())
        assert torch.equal(y.view(n, heads, d)[..., r:], x.view(n, heads, d)[..., r:])      # the rest is copied


@pytest.mark.parametrize("dtype,pad", [("f32", 0), ("bf16", 0), ("f16", 1), ("f32", 1), ("bf16", 2)])
def test_rope_append_from_fused_rows(dtype, pad):
    """q, k, v of one fused row (rows `pad` elements longer, so that they start
    at any alignment) into q rows and cache slots; -1 and n_rows skip a token."""
    tid, dt = R.TYPES[dtype]
    n, H, kv, d, r, rows = 37, 6, 2, 64, 48, 100
    g = _gen(3)
    qkv = _randn(g, dt, n, (H + 2 * kv) * d + pad)
    q, k, v = qkv[:, pad:pad + H * d], qkv[:, pad + H * d:pad + (H + kv) * d], qkv[:, pad + (H + kv) * d:]
    qo = torch.full((n, H * d + pad), NAN, dtype=dt, device="cuda")
    ko, vo = _randn(g, dt, rows, kv * d), _randn(g, dt, rows, kv * d)
    k0, v0 = ko.clone(), vo.clone()
    slots = torch.randperm(rows, generator=g, device="cuda")[:n].to(torch.int32)
    slots[3], slots[20] = -1, rows
    pos = torch.arange(100, 100 + n, device="cuda", dtype=torch.int32)
    R.rope(R.rope_args(tid, q, k, v, qo[:, :H * d], ko, vo, n_tokens=n, n_heads=H, n_kv_heads=kv, head_dim=d,
                       rope_dim=r, positions=pos, theta=1e4, slots=R.ptr(slots), n_rows=rows))
    ang, gain = R.rope_angles(pos, r, 1e4)
    want, mass = R.rope_ref(q.reshape(n, H, d), ang, gain, r, 0)
    assert ((qo[:, :H * d].reshape(n, H, d).double().cpu() - want).abs() <= _rope_tol(mass, want, dt)).all()
    assert qo[:, H * d:].isnan().all()
    want, mass = R.rope_ref(k.reshape(n, kv, d), ang, gain, r, 0)
    ok = torch.tensor([0 <= s < rows for s in slots.tolist()])
    at = slots.cpu()[ok].long()
    got = ko.cpu()[at].double().view(-1, kv, d)
    assert ((got - want[ok]).abs() <= _rope_tol(mass, want, dt)[ok]).all()
    assert torch.equal(vo.cpu()[at], v.cpu()[ok])
    others = torch.ones(rows, dtype=torch.bool)
    others[at] = False
    assert torch.equal(ko.cpu()[others], k0.cpu()[others]) and torch.equal(vo.cpu()[others], v0.cpu()[others])


@pytest.mark.parametrize("ilv", [0, 1])
def test_rope_in_place_and_back(ilv):
    """In place gives the bits of out of place; the inverse gives x back (two
    rotations, so twice the tolerance, counted on the pair's mass)."""
    n, H, d, r = 50, 4, 128, 64
    g = _gen(9)
    x = _randn(g, torch.float32, n, H * d)
    pos = torch.randint(0, 1 << 20, (n,), generator=g, device="cuda", dtype=torch.int32)
    kw = dict(n_tokens=n, n_heads=H, n_kv_heads=0, head_dim=d, rope_dim=r, positions=pos, theta=1e6, layout=ilv)
    y = torch.empty_like(x)
    R.rope(R.rope_args(0, x, None, None, y, **kw))
    z = x.clone()
    R.rope(R.rope_args(0, z, None, None, z, **kw))
    assert torch.equal(y, z)
    R.rope(R.rope_args(0, z, None, None, z, inverse=1, **kw))
    ang, gain = R.rope_angles(pos, r, 1e6)
    _, mass = R.rope_ref(x.view(n, H, d), ang, gain, r, ilv)
    # the second rotation sees values of up to mass and errors of the first
    assert ((z - x).view(n, H, d).double().cpu().abs() <= 4 * mass * 2.0 ** -21 + 1e-30).all()


def test_rope_inverse_is_the_gradient():
    """d(sum w . rope(x)) / dx = rope_inverse(w), against central differences of
    the plain form (linear in x, so exact up to fp64 rounding)."""
    n, H, d, r = 3, 2, 16, 8
    g = _gen(1)
    w = _randn(g, torch.float32, n, H * d)
    pos = torch.tensor([0, 5, 90000], dtype=torch.int32, device="cuda")
    got = torch.empty_like(w)
    R.rope(R.rope_args(0, w, None, None, got, n_tokens=n, n_heads=H, n_kv_heads=0, head_dim=d, rope_dim=r, positions=pos,
                       theta=1e4, inverse=1))
    ang, gain = R.rope_angles(pos, r, 1e4)
    wd = w.double().cpu().view(n, H, d)
    want = torch.zeros(n, H, d, dtype=torch.float64)
    for i in range(d):
        x = torch.zeros(n, H, d, dtype=torch.float64)
        x[..., i] = 1.0
        up, down = R.rope_ref(x, ang, gain, r, 0)[0], R.rope_ref(-x, ang, gain, r, 0)[0]
        want[..., i] = ((up - down) / 2 * wd).sum(-1)
    _, mass = R.rope_ref(wd, ang, gain, r, 0)
    assert ((got.double().cpu().view(n, H, d) - want).abs() <= _rope_tol(mass, want, torch.float32)).all()


def test_rope_freq_factors_and_fused_out():
    """Per-pair factors; q_out and k_out as slices of one fused row."""
    n, H, kv, d, r = 9, 2, 1, 32, 32
    g = _gen(4)
    x = _randn(g, torch.float32, n, (H + kv) * d)
    y = torch.full_like(x, NAN)
    ff = torch.rand(r // 2, generator=g, device="cuda") + 0.5
    pos = torch.arange(n, device="cuda", dtype=torch.int32) * 1000
    R.rope(R.rope_args(0, x[:, :H * d], x[:, H * d:], None, y[:, :H * d], y[:, H * d:], n_tokens=n, n_heads=H,
                       n_kv_heads=kv, head_dim=d, rope_dim=r, positions=pos, theta=1e4, scaling=1, factor=2.0,
                       freq_factors=R.ptr(ff)))
    ang, gain = R.rope_angles(pos, r, 1e4, scaling=1, factor=2.0, freq_factors=ff)
    want, mass = R.rope_ref(x.view(n, H + kv, d), ang, gain, r, 0)
    assert ((y.view(n, H + kv, d).double().cpu() - want).abs() <= _rope_tol(mass, want, torch.float32)).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attn_case(dtype, B, T, H, kv, d, P, L, lens, seed=0, weights=False, pad=0):
    """Tensors with padded strides, garbage in every row that is not to be read."""
    tid, dt = R.TYPES[dtype]
    g = _gen(seed + 17)
    q = (_randn(g, dt, B, T, H + 2 * pad, d) * 2)[:, :, :H]
    c = dict(q=q, out=torch.full((B, T, H + pad, d), NAN, dtype=dt, device="cuda")[:, :, :H])
    if P:
        c["pk"], c["pv"] = _randn(g, dt, P, kv, d), _randn(g, dt, P, kv, d)
    if L:
        c["k"], c["v"] = _randn(g, dt, B, L + pad, kv, d), _randn(g, dt, B, L + pad, kv, d)
        c["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for b, n in enumerate(lens):
            n = max(0, min(n, L))
            c["k"][b, n:], c["v"][b, n:] = NAN, float("inf")
        if weights:
            c["scores"] = torch.rand(B, kv, L + pad, generator=g, device="cuda")
    return tid, c, (L or None)


def _check_attn(tid, c, L, scale=0.0, ws=None):
    before = c["scores"].clone() if "scores" in c else None
    R.attention(R.attention_args(tid, max_len=L, scale=scale, **c), ws)
    out, tol, gathered, gtol = R.attention_ref(c["q"], c.get("lens"), c.get("k"), c.get("v"), c.get("pk"), c.get("pv"),
                                               scale, L)
    err = (c["out"].double() - out).abs()
    assert (err <= tol).all(), f"worst error / tolerance {float((err / tol).max())}"
    if before is not None:
        got = c["scores"].double()
        want = before.double()
        want[..., :L] += gathered
        err = (got - want).abs()[..., :L]
        lim = gtol + want[..., :L].abs() * 2.0 ** -24
        assert (err <= lim).all(), f"worst weight error / tolerance {float((err / lim).max())}"
        for b, n in enumerate(c["lens"].tolist()):
            n = max(0, min(n, L))
            assert torch.equal(c["scores"][b, :, n:], before[b, :, n:])


ATTN = [
    # type, batch, tokens, heads, kv, dim, prefix, max_len, lens
    ("f32", 1, 1, 8, 2, 256, 0, 1, [1]),                             # one row
    ("f32", 1, 1, 8, 2, 256, 0, 40, [0]),                            # none: zeros
    ("f32", 4, 1, 8, 2, 256, 500, 12, [0, 1, 12, 7]),
    ("f32", 3, 1, 16, 4, 256, 2048, 300, [300, 17, 129]),
    ("f32", 9, 2, 8, 2, 64, 333, 20, [2, 1, 0, 20, 5, 19, 16, 17, 18]),   # 72 prefix rows per KV head
    ("f32", 2, 3, 15, 3, 128, 65, 1000, [1000, 2]),                  # group 5; a token that sees no own row
    ("f32", 5, 8, 5, 1, 128, 100, 90, [90, 40, 8, 3, 0]),            # 40 own rows: a row tile of the CTA is empty
    ("f32", 7, 8, 4, 1, 256, 300, 40, [40] * 7),                     # 224 prefix rows
    ("bf16", 1, 1, 1, 1, 64, 1, 0, []),
    ("bf16", 5, 1, 16, 2, 128, 1000, 333, [333, 0, 128, 129, 1]),
    ("bf16", 33, 1, 8, 2, 256, 513, 33, list(range(33))),            # 132 prefix rows per KV head
    ("bf16", 2, 1, 32, 8, 128, 0, 5001, [5001, 4097]),
    ("f16", 5, 4, 12, 4, 64, 1000, 333, [333, 4, 3, 200, 0]),
    ("f16", 1, 70, 4, 2, 64, 31, 129, [129]),                        # 140 own rows per KV head
    ("f16", 40, 2, 8, 1, 128, 700, 40, [(7 * i) % 41 for i in range(40)]),   # 640 prefix rows
    ("bf16", 3, 1, 4, 4, 128, 257, 50, [60, -3, 50]),                # lens outside [0, max_len] are clamped
    ("f16", 2, 1, 16, 1, 256, 4097, 100, [100, 99]),
    ("bf16", 17, 8, 8, 1, 64, 1, 9, [9] * 17),
    ("f16", 1, 1, 16, 4, 128, 40001, 5, [5]),                        # four query rows on a long prefix
    ("bf16", 3, 1, 12, 4, 64, 100001, 5, [5, 1, 0]),
    ("bf16", 17, 1, 4, 4, 128, 9001, 5, [5, 1, 0] * 5 + [2, 2]),     # 17 prefix rows per KV head
    ("f16", 5, 1, 16, 4, 64, 60001, 70, [70, 64, 1, 65, 0]),
    ("bf16", 65, 1, 16, 4, 64, 4097, 3, [3] * 65),                   # 260 prefix rows, the last four in a tile of their own
]


@pytest.mark.parametrize("dtype,B,T,H,kv,d,P,L,lens", ATTN)
def test_attention(dtype, B, T, H, kv, d, P, L, lens):
    _check_attn(*_attn_case(dtype, B, T, H, kv, d, P, L, lens))


WEIGHTS = [
    ("f32", 1, 1, 8, 2, 256, 0, 500, [500]),
    ("f32", 3, 2, 6, 2, 64, 100, 300, [300, 0, 129]),                # weights of own rows beside a prefix
    ("bf16", 4, 1, 32, 8, 128, 0, 700, [700, 1, 699, 300]),
    ("f16", 2, 5, 4, 1, 128, 0, 260, [260, 3]),                      # tokens that see nothing
    ("bf16", 1, 80, 2, 2, 64, 0, 200, [200]),                        # more query rows than one pass of statistics
]


@pytest.mark.parametrize("dtype,B,T,H,kv,d,P,L,lens", WEIGHTS)
def test_attention_gathers_weights(dtype, B, T, H, kv, d, P, L, lens):
    _check_attn(*_attn_case(dtype, B, T, H, kv, d, P, L, lens, weights=True))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_strides_scale_and_gaps(dtype):
    """Padded token rows, slices and score rows; the gaps stay as they were; an
    explicit scale; out written over q."""
    tid, c, L = _attn_case(dtype, 3, 2, 4, 2, 64, 130, 77, [77, 5, 40], weights=True, pad=3)
    whole = c["out"]._base if c["out"]._base is not None else c["out"]
    _check_attn(tid, c, L, scale=0.3)
    assert whole[:, :, 4:].isnan().all()
    want = c["out"].clone()
    c2 = {n: x for n, x in c.items() if n != "scores"}
    c2["out"] = c2["q"]
    R.attention(R.attention_args(tid, max_len=L, scale=0.3, **c2))
    assert torch.equal(c2["q"], want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_extremes(dtype):
    """Logits far apart (one row takes all the weight, others underflow) and
    equal (all rows share it), of large size."""
    tid, c, L = _attn_case(dtype, 2, 1, 4, 2, 128, 300, 200, [200, 100], weights=True)
    c["q"].mul_(20)
    _check_attn(tid, c, L)
    c["q"].zero_()
    _check_attn(tid, c, L)
    c["pk"].fill_(1.0)
    c["k"][:, :100].fill_(1.0)
    c["q"].fill_(30.0)
    _check_attn(tid, c, L)


@pytest.mark.parametrize("dtype,kv,d,scale,P", [("bf16", 1, 128, 0.0, 3000), ("f16", 2, 64, -0.4, 3000),
                                                ("bf16", 1, 256, 0.1, 3000), ("f16", 4, 64, 0.0, 6001),
                                                ("bf16", 4, 64, -0.2, 6017)])
def test_attention_prefix_maximum_rises(dtype, kv, d, scale, P):
    """Many query rows on a prefix whose logits grow along it, so that the running
    maximum rises by far more than the slack again and again, in some rows only."""
    tid, c, L = _attn_case(dtype, 24, 2, 4 * kv, kv, d, P, 40, [40 - b for b in range(24)])
    c["pk"] *= torch.linspace(0.05, 6, P, device="cuda")[:, None, None].to(c["pk"].dtype)
    c["q"][::3] *= 0.01
    _check_attn(tid, c, L, scale)
    assert lib().inferno_device_error(0, 0) == 0


def test_attention_nan_rows_stay_apart():
    """A NaN in one sequence's rows makes that sequence's heads NaN, no others."""
    tid, c, L = _attn_case("bf16", 3, 1, 4, 2, 64, 100, 60, [60, 60, 60])
    c["k"][1, 30, 0] = NAN
    c["q"][2, 0, 3] = NAN
    R.attention(R.attention_args(tid, max_len=L, **c))
    nan = c["out"].isnan()
    assert nan[1, 0, :2].all() and not nan[1, 0, 2:].any()
    assert nan[2, 0, 3].all() and not nan[2, 0, :3].any() and not nan[0].any()


@pytest.mark.parametrize("dtype,H,d,T", [("f32", 1, 256, 4), ("f32", 2, 128, 2), ("f32", 3, 64, 5), ("f32", 6, 256, 5),
                                         ("bf16", 2, 128, 3), ("f16", 8, 64, 4), ("bf16", 4, 256, 20)])
def test_attention_padded_tokens(dtype, H, d, T):
    """The rows of the last tokens hold garbage (padding): the tokens before them
    get what they get from clean rows, bit for bit, those that see them NaN."""
    tid, c, L = _attn_case(dtype, 3, T, 2 * H, 2, d, 40, 90, [90, 33, T], seed=4, weights=True)
    clean = {n: x.clone() if n in ("out", "scores") else x for n, x in c.items()}
    R.attention(R.attention_args(tid, max_len=L, **clean))
    for b, n in enumerate([90, 33, T]):
        c["k"][b, n - 1], c["v"][b, n - 1] = NAN, float("inf")
    R.attention(R.attention_args(tid, max_len=L, **c))
    assert torch.equal(c["out"][:, :-1], clean["out"][:, :-1])
    assert c["out"][:, -1].isnan().all()


def test_attention_repeats_bit_for_bit():
    for dtype, P in (("f32", 700), ("bf16", 3001)):
        tid, c, L = _attn_case(dtype, 40, 1, 8, 2, 128, P, 300, [(13 * i) % 301 for i in range(40)])
        a = R.attention_args(tid, max_len=L, **c)
        R.attention(a)
        first = c["out"].clone()
        ws = R.attention_workspace(a).fill_(0xFF)           # a workspace needs no initialisation
        for _ in range(3):
            R.attention(a, ws)
            assert torch.equal(c["out"], first)
        assert lib().inferno_device_error(0, 0) == 0


def test_attention_captured_reads_lengths_on_the_device():
    tid, c, L = _attn_case("bf16", 6, 1, 8, 2, 128, 900, 200, [200] * 6, weights=True)
    a = R.attention_args(tid, max_len=L, **c)
    ws = R.attention_workspace(a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        R.attention(a, ws)
    for lens in ([200, 1, 0, 50, 199, 128], [0] * 6, [3, 200, 200, 17, 16, 15]):
        c["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        c["scores"].zero_()
        c["out"].fill_(NAN)
        graph.replay()
        out, tol, gathered, gtol = R.attention_ref(c["q"], lens, c["k"], c["v"], c["pk"], c["pv"], 0.0, L)
        assert ((c["out"].double() - out).abs() <= tol).all()
        assert ((c["scores"].double() - gathered).abs() <= gtol + gathered * 2.0 ** -24).all()


def test_attention_on_two_streams():
    """Calls on two streams at once, a workspace each, give the bits of calls alone."""
    cases = [_attn_case("bf16", 8, 1, 16, 2, 128, 4000, 400, [400] * 8, seed=s) for s in (1, 2)]
    args = [R.attention_args(t, max_len=L, **c) for t, c, L in cases]
    want = []
    for a, (_, c, _) in zip(args, cases):
        R.attention(a)
        want.append(c["out"].clone())
    ws = [R.attention_workspace(a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    for _ in range(10):
        for a, w, s in zip(args, ws, streams):
            with torch.cuda.stream(s):
                R.attention(a, w)
    torch.cuda.synchronize()
    for (_, c, _), w in zip(cases, want):
        assert torch.equal(c["out"], w)


def test_attention_far_offsets():
    """Slices whose element offsets pass 2^31."""
    stride = (1 << 31) // 64 * 64 + 4096
    k = torch.empty(stride + 8 * 64, dtype=torch.float16, device="cuda")
    v = torch.empty(stride + 8 * 64, dtype=torch.float16, device="cuda")
    g = _gen(5)
    c = dict(q=_randn(g, torch.float16, 2, 1, 2, 64), out=torch.empty(2, 1, 2, 64, dtype=torch.float16, device="cuda"),
             lens=torch.tensor([8, 5], dtype=torch.int32, device="cuda"))
    ks, vs = (torch.as_strided(x, (2, 8, 1, 64), (stride, 64, 64, 1)) for x in (k, v))
    for x in (ks, vs):
        x.copy_(_randn(g, torch.float16, 2, 8, 1, 64))
    _check_attn(1, dict(c, k=ks, v=vs), 8)


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------
def _evict_case(dtype, B, kv, d, rows, seed=0):
    tid, dt = R.TYPES[dtype]
    g = _gen(seed + 5)
    k, v = _randn(g, dt, B, rows, kv, d), _randn(g, dt, B, rows, kv, d)
    scores = torch.rand(B, kv, rows, generator=g, device="cuda")
    pos = torch.rand(B, kv, rows, generator=g, device="cuda").argsort(-1).to(torch.int32)
    return tid, k, v, scores, pos


def _check_evict(tid, k, v, scores, pos, lens, next_pos, in_place=False, **kw):
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    nxt = torch.tensor(next_pos, dtype=torch.int32, device="cuda")
    so = scores if in_place else torch.full_like(scores, -7.0)
    po = pos if in_place else torch.full_like(pos, -7)
    lo = lens if in_place else torch.full_like(lens, -7)
    want = R.evict_ref(k, v, scores, pos, lens.tolist(), nxt, so, po, **kw)
    R.evict(R.evict_args(tid, k, v, scores, pos, lens, nxt, so, po, lo, **kw))
    for name, got, w in zip(("k", "v", "scores", "slot_pos", "lens"), (k, v, so, po, lo), want):
        same = (got.cpu() == w) | (got.cpu().isnan() & w.isnan())
        assert same.all(), f"{name}: {int((~same).sum())} of {same.numel()} differ"


EVICT = [
    # type, batch, kv, dim, rows, lens, budget, sink, recent
    ("f32", 1, 1, 64, 2, [2], 1, 0, 0),
    ("f32", 2, 2, 256, 65, [65, 64], 64, 4, 16),                     # one row over the budget; none over
    ("bf16", 3, 2, 128, 1500, [1500, 1025, 3], 1024, 4, 100),
    ("f16", 2, 3, 64, 2100, [2100, 700], 100, 1, 99),                # every kept row is a sink or recent
    ("bf16", 1, 2, 8, 3000, [3000], 2999, 0, 0),
    ("f32", 1, 1, 4, 5000, [5000], 1, 0, 1),
    ("f16", 4, 1, 80, 300, [0, -5, 400, 300], 150, 2, 10),           # lens are clamped
    ("f32", 2, 1, 128, 6000, [6000, 2500], 3000, 4, 700),            # more to move than the clusters take
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype,B,kv,d,rows,lens,budget,sink,recent", EVICT)
def test_evict(dtype, B, kv, d, rows, lens, budget, sink, recent, in_place):
    tid, k, v, scores, pos = _evict_case(dtype, B, kv, d, rows)
    _check_evict(tid, k, v, scores, pos, lens, [max(n, 0) for n in lens], in_place, budget=budget, n_sink=sink,
                 n_recent=recent)


@pytest.mark.parametrize("kind", ["equal", "few values", "zeros of both signs", "nan and infinities", "subnormal", "negative"])
def test_evict_ties_and_odd_scores(kind):
    tid, k, v, scores, pos = _evict_case("bf16", 2, 2, 64, 2500, seed=3)
    g = _gen(8)
    pick = torch.randint(0, 4, scores.shape, generator=g, device="cuda")
    values = {"equal": [1.0] * 4, "few values": [0.0, 1.0, 2.0, 1.0], "zeros of both signs": [0.0, -0.0, 0.0, 1.0],
              "nan and infinities": [NAN, float("inf"), -float("inf"), 1.0], "subnormal": [1e-42, 2e-42, 0.0, 1e-45],
              "negative": [-1.0, -2.0, 0.5, -3e38]}[kind]
    scores.copy_(torch.tensor(values, device="cuda")[pick])
    _check_evict(tid, k, v, scores, pos, [2500, 2049], [2500, 2500], budget=1300, n_sink=3, n_recent=50)


@pytest.mark.parametrize("rows", [2000, 20000])
@pytest.mark.parametrize("bit", [0, 7, 8, 15, 16, 22, 23, 26, 31])
@pytest.mark.parametrize("short", [0, 1, -1])
def test_evict_border_between_two_values(rows, bit, short):
    """Scores of two values that differ in one bit, as many of the larger as the
    budget holds, one more and one fewer."""
    tid, k, v, scores, pos = _evict_case("f16", 1, 2, 8, rows, seed=bit)
    hi = rows // 3
    low = 0x3a000000
    bits = torch.full(scores.shape, low, dtype=torch.int64, device="cuda")
    for h in range(2):
        at = torch.randperm(rows, generator=_gen(bit + 40 + h), device="cuda")[:hi]
        bits[0, h, at] = low ^ (1 << bit)
    if bit == 31 or low & (1 << bit):          # the changed value is the smaller one
        hi = rows - hi
    scores.copy_(torch.where(bits >= 2**31, bits - 2**32, bits).to(torch.int32).view(torch.float32))
    _check_evict(tid, k, v, scores, pos, [rows], [rows], budget=hi + short, n_sink=0, n_recent=0)


def test_evict_more_kept_always_than_budget():
    """Positions named twice can put more rows under protection than the budget
    holds: they are then ranked by score."""
    tid, k, v, scores, pos = _evict_case("f32", 1, 1, 16, 1200, seed=6)
    pos.fill_(0)
    _check_evict(tid, k, v, scores, pos, [1200], [1200], budget=300, n_sink=1, n_recent=0)


@pytest.mark.parametrize("rows,budget,d", [(40000, 9000, 8), (30000, 12000, 256), (800000, 100000, 8)])
def test_evict_long(rows, budget, d):
    """Parts of a cluster that hold their keys in shared memory, rows that a second
    kernel moves, and parts too long for shared memory."""
    tid, k, v, scores, pos = _evict_case("bf16", 1, 1, d, rows, seed=7)
    _check_evict(tid, k, v, scores, pos, [rows - 3], [rows], budget=budget, n_sink=4, n_recent=budget // 3)


def test_evict_strides_and_max_len():
    tid, dt = R.TYPES["f16"]
    g = _gen(2)
    big, bigv = _randn(g, dt, 2, 200, 2, 32), _randn(g, dt, 2, 200, 2, 32)
    scores = torch.rand(2, 2, 210, generator=g, device="cuda")
    pos = torch.rand(2, 2, 210, generator=g, device="cuda").argsort(-1).to(torch.int32)
    _check_evict(tid, big, bigv, scores, pos, [180, 190], [210, 210], budget=90, n_sink=0, n_recent=20, max_len=180)


def test_evict_captured():
    tid, k, v, scores, pos = _evict_case("bf16", 3, 2, 64, 600)
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    nxt = torch.full((3,), 600, dtype=torch.int32, device="cuda")
    a = R.evict_args(tid, k, v, scores, pos, lens, nxt, scores, pos, lens, budget=256, n_sink=2, n_recent=9)
    ws = R.evict_workspace(a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        R.evict(a, ws)
    for n in ([600, 257, 256], [400, 0, 599]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        scores.uniform_()
        want = R.evict_ref(k, v, scores, pos, n, nxt, scores, pos, budget=256, n_sink=2, n_recent=9)
        graph.replay()
        for got, w in zip((k, v, scores, pos, lens), want):
            assert torch.equal(got.cpu(), w)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decode_steps_with_a_shared_prefix_and_a_budget(dtype):
    """Sequences on one prefix decode: q and k are rotated and appended, attend to
    prefix and own rows, the weights gather, and a cache that has grown 8 rows over
    its budget is cut back.  Each call is checked on its own inputs."""
    tid, dt = R.TYPES[dtype]
    B, H, kv, d, r, P, budget, slack = 3, 8, 2, 64, 32, 150, 24, 8
    rows = budget + slack
    g = _gen(12)
    pk, pv = _randn(g, dt, P, kv, d), _randn(g, dt, P, kv, d)
    k, v = torch.full((B, rows, kv, d), NAN, dtype=dt, device="cuda"), torch.full((B, rows, kv, d), NAN, dtype=dt, device="cuda")
    scores = torch.zeros(B, kv, rows, device="cuda")
    pos = torch.zeros(B, kv, rows, dtype=torch.int32, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    nxt = torch.full((B,), P, dtype=torch.int32, device="cuda")
    first = torch.arange(B, device="cuda", dtype=torch.int32) * rows
    evictions = 0
    for step in range(50):
        qkv = _randn(g, dt, B, (H + 2 * kv) * d)
        q = torch.empty(B, 1, H, d, dtype=dt, device="cuda")
        slots = first + lens
        R.rope(R.rope_args(tid, qkv[:, :H * d], qkv[:, H * d:(H + kv) * d], qkv[:, (H + kv) * d:], q.view(B, H * d),
                           k.view(B * rows, kv * d), v.view(B * rows, kv * d), n_tokens=B, n_heads=H, n_kv_heads=kv,
                           head_dim=d, rope_dim=r, positions=nxt, theta=1e4, slots=R.ptr(slots), n_rows=B * rows))
        ang, gain = R.rope_angles(nxt, r, 1e4)
        want, mass = R.rope_ref(qkv[:, H * d:(H + kv) * d].reshape(B, kv, d), ang, gain, r, 0)
        got = k.view(B * rows, kv, d)[slots.long()].double().cpu()
        assert ((got - want).abs() <= _rope_tol(mass, want, dt)).all()
        at = lens.long()[:, None, None].expand(B, kv, 1)
        scores.scatter_(2, at, 0.0)
        pos.scatter_(2, at, nxt[:, None, None].expand(B, kv, 1))
        lens += 1
        nxt += 1
        out = torch.empty_like(q)
        _check_attn(tid, dict(q=q, out=out, pk=pk, pv=pv, k=k, v=v, lens=lens, scores=scores), rows)
        if int(lens.max()) == rows:
            evictions += 1
            n = lens.tolist()
            want = R.evict_ref(k, v, scores, pos, n, nxt, scores, pos, budget=budget, n_recent=6)
            R.evict(R.evict_args(tid, k, v, scores, pos, lens, nxt, scores, pos, lens, budget=budget, n_recent=6))
            for x, w in zip((k, v, scores, pos, lens), want):
                same = (x.cpu() == w) | (x.cpu().isnan() & w.isnan())
                assert same.all()
    assert evictions >= 3
    assert lib().inferno_device_error(0, 1) == 0


def test_first_calls_may_be_captured():
    """A process whose first calls are made under capture."""
    import subprocess
    import sys
    code = """
import sys
sys.path[:0] = [%r, %r]
import torch, longctx_ref as R
B, H, d = 40, 4, 128
q = torch.randn(B, 1, H, d, device="cuda", dtype=torch.bfloat16)
k, v = (torch.randn(B, 64, 2, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
pk, pv = (torch.randn(1000, 2, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
lens = torch.full((B,), 60, dtype=torch.int32, device="cuda")
scores, pos = torch.zeros(B, 2, 64, device="cuda"), torch.zeros(B, 2, 64, dtype=torch.int32, device="cuda")
out = torch.empty_like(q)
a = R.attention_args(30, q, out, lens, k, v, pk, pv, scores)
e = R.evict_args(30, k, v, scores, pos, lens, lens, scores, pos, lens, budget=32)
wa, we = R.attention_workspace(a), R.evict_workspace(e)
at = torch.zeros(B, dtype=torch.int32, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    R.rope(R.rope_args(30, q.view(B, -1), None, None, q.view(B, -1), n_tokens=B, n_heads=H, n_kv_heads=0, head_dim=d,
                       rope_dim=d, positions=at, theta=1e4))
    R.attention(a, wa)
    R.evict(e, we)
g.replay()
print("lens", lens.unique().tolist(), "finite", bool(out.isfinite().all()))
""" % (str(R.__file__).rsplit("/", 1)[0], str(R.InfernoRope.__module__ and __import__("inferno_b200").__path__[0]).rsplit("/", 1)[0])
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert "lens [32] finite True" in out.stdout, out.stdout + out.stderr[-2000:]


def test_host_memory_is_refused():
    host = torch.zeros(64, dtype=torch.float32)
    dev = torch.zeros(64, device="cuda")
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    a = R.rope_args(0, dev[None], None, None, host[None], n_tokens=1, n_heads=1, n_kv_heads=0, head_dim=64, rope_dim=64,
                    positions=pos, theta=1e4)
    with pytest.raises(InfernoError, match="not device memory"):
        call("inferno_rope", C.byref(a), R.stream())
