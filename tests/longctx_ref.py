"""Plain 64-bit forms of the long-context operators (inferno_rope,
inferno_attention_cached, inferno_cache_evict) and calls of the library on torch
tensors, shared by their tests."""
import ctypes as C
import math

import torch

from inferno_b200._lib import InfernoAttention, InfernoEvict, InfernoRope, call, lib

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def ptr(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def rope_angles(positions, rope_dim, theta, scaling=0, factor=1.0, orig_ctx=4096, beta_fast=32.0, beta_slow=1.0,
                mscale=0.0, freq_factors=None):
    """(angles [tokens][pairs], factor of cos and sin) in float64."""
    i = torch.arange(rope_dim // 2, dtype=torch.float64)
    f = theta ** (-2.0 * i / rope_dim)
    if freq_factors is not None:
        f = f / freq_factors.double().cpu()
    gain = mscale if mscale else 1.0
    if scaling == 1:
        f = f / factor
    elif scaling == 2:
        d = [rope_dim * math.log(orig_ctx / (2 * math.pi * n)) / (2 * math.log(theta)) for n in (beta_fast, beta_slow)]
        low, high = max(math.floor(d[0]), 0), min(math.ceil(d[1]), rope_dim - 1)
        r = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f * (1 - r) + f / factor * r
        if not mscale and factor > 1:
            gain = 0.1 * math.log(factor) + 1
    return positions.cpu().double()[:, None] * f, gain


def rope_ref(x, angles, gain, rope_dim, interleaved, inverse=False):
    """x [tokens][heads][dim] -> rotated in float64; also sum of |a| + |b| of each value's pair."""
    y = x.double().cpu().clone()
    half = rope_dim // 2
    ia = torch.arange(0, rope_dim, 2) if interleaved else torch.arange(half)
    ib = ia + 1 if interleaved else ia + half
    c, s = (angles.cos() * gain)[:, None], (angles.sin() * gain * (-1 if inverse else 1))[:, None]
    a, b = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    mass = torch.zeros_like(y)
    mass[..., ia] = mass[..., ib] = (a.abs() + b.abs()) * gain
    return y, mass


def rope_args(type_id, q=None, k=None, v=None, q_out=None, k_out=None, v_out=None, *, n_tokens, n_heads, n_kv_heads,
              head_dim, rope_dim, positions, **kw):
    a = InfernoRope(type=type_id, n_tokens=n_tokens, n_heads=n_heads, n_kv_heads=n_kv_heads, head_dim=head_dim,
                    rope_dim=rope_dim, positions=ptr(positions), **kw)
    for name, t in (("q", q), ("k", k), ("v", v), ("q_out", q_out), ("k_out", k_out), ("v_out", v_out)):
        if t is not None:
            setattr(a, name, t.data_ptr())
            setattr(a, name + "_stride", t.stride(0))
    return a


def rope(a):
    return call("inferno_rope", C.byref(a), stream())


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def attention_args(type_id, q, out, lens=None, k=None, v=None, pk=None, pv=None, scores=None, max_len=None, scale=0.0):
    """q, out [batch][tokens][heads][dim] (dim and heads contiguous); k, v
    [batch][rows][kv][dim]; pk, pv [rows][kv][dim]."""
    B, T, H, d = q.shape
    kv = (k if k is not None else pk).shape[-2]
    a = InfernoAttention(type=type_id, batch=B, n_tokens=T, n_heads=H, n_kv_heads=kv, head_dim=d, scale=scale,
                         q=ptr(q), out=ptr(out), q_stride=q.stride(1), out_stride=out.stride(1))
    if pk is not None:
        a.prefix_len, a.prefix_k, a.prefix_v = pk.shape[0], ptr(pk), ptr(pv)
    if k is not None:
        a.max_len, a.k_cache, a.v_cache, a.lens = max_len or k.shape[1], ptr(k), ptr(v), ptr(lens)
        a.seq_stride = k.stride(0)
    if scores is not None:
        a.scores, a.score_stride = ptr(scores), scores.stride(1)
    return a


def attention_workspace(a):
    return torch.empty(call("inferno_attention_cached_workspace", C.byref(a)), dtype=torch.uint8, device="cuda")


def attention(a, ws=None):
    ws = attention_workspace(a) if ws is None else ws
    call("inferno_attention_cached", C.byref(a), C.c_void_p(ws.data_ptr()), ws.numel(), stream())


def attention_ref(q, lens, k, v, pk=None, pv=None, scale=0.0, max_len=None):
    """float64: out, gathered weight [batch][kv][rows], and their error bounds.

    The bounds count roundings.  A logit of hd products is off by at most
    delta = scale * sum |q||k| * e, e = hd 2^-24 for the fp32 sum, plus for fp32
    operands 2^-19 for the pair products (hi has 11 bits, so |lo| <= 2^-11 |x|;
    lo is read to 11 bits, 2^-21 |x| for either factor, lo lo <= 2^-22 is dropped:
    below 2^-19.6 together); the products with V add the same once more.  exp2 adds
    2^-22, its fp32 argument |logit| 2^-22 (scale, log2 e, their product with the
    sum, the largest taken off: 2^-24 each).
    Every weight and their sum is then off by that relative amount, the sums over
    n rows by (n + 64) 2^-24; the 16-bit types round each weight (before the
    product with V) and the output, half a step each."""
    B, T, H, d = q.shape
    kv = (k if k is not None else pk).shape[-2]
    G, dt = H // kv, q.dtype
    scale = scale or d ** -0.5
    rows = 0 if k is None else (max_len or k.shape[1])
    out = torch.zeros(B, T, H, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    gathered = torch.zeros(B, kv, rows, dtype=torch.float64, device=q.device)
    gtol = torch.zeros_like(gathered)
    u = half_step(dt)
    pair = 2.0 ** -19 if dt == torch.float32 else 0.0
    e = d * 2.0 ** -24 + pair
    P = 0 if pk is None else pk.shape[0]
    for b in range(B):
        n = 0 if k is None else max(0, min(int(lens[b]), rows))
        for h in range(kv):
            keys = torch.cat([x.double() for x in ([pk[:, h]] if P else []) + ([k[b, :n, h]] if n else [])]) if P + n else None
            vals = torch.cat([x.double() for x in ([pv[:, h]] if P else []) + ([v[b, :n, h]] if n else [])]) if P + n else None
            for t in range(T):
                seen = P + max(0, n - T + 1 + t)
                if not seen:
                    continue
                x = q[b, t, h * G:(h + 1) * G].double()
                s = x @ keys[:seen].t() * scale
                delta = (x.abs() @ keys[:seen].abs().t() * abs(scale) * e).amax(-1, keepdim=True)
                p = torch.softmax(s, -1)
                # numerator and denominator
                rel = 2 * (delta + 2.0 ** -22 + s.abs().amax(-1, keepdim=True) * 2.0 ** -22) + (seen + 64) * 2.0 ** -23
                o, mass = p @ vals[:seen], p @ vals[:seen].abs()
                out[b, t, h * G:(h + 1) * G] = o
                # the last term: values below the normal range round absolutely
                tol[b, t, h * G:(h + 1) * G] = (mass * (rel + (u if dt != torch.float32 else pair)) * 1.01 + o.abs() * u
                                                + torch.finfo(dt).smallest_normal)
                gathered[b, h, :seen - P] += p[:, P:].sum(0)
                gtol[b, h, :seen - P] += (p[:, P:] * (rel + (G * T + 2) * 2.0 ** -24)).sum(0) + 2.0 ** -126
    return out, tol, gathered, gtol


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------
def evict_args(type_id, k, v, scores, pos, lens, next_pos, scores_out, pos_out, lens_out, *, budget, n_sink=0,
               n_recent=0, max_len=None):
    B, rows, kv, d = k.shape
    return InfernoEvict(type=type_id, batch=B, n_kv_heads=kv, head_dim=d, max_len=max_len or rows, budget=budget,
                        n_sink=n_sink, n_recent=n_recent, seq_stride=k.stride(0), score_stride=scores.stride(1),
                        k_cache=ptr(k), v_cache=ptr(v), scores=ptr(scores), slot_pos=ptr(pos), lens=ptr(lens),
                        next_pos=ptr(next_pos), scores_out=ptr(scores_out), slot_pos_out=ptr(pos_out),
                        lens_out=ptr(lens_out))


def evict_workspace(a):
    return torch.empty(call("inferno_cache_evict_workspace", C.byref(a)), dtype=torch.uint8, device="cuda")


def evict(a, ws=None):
    ws = evict_workspace(a) if ws is None else ws
    call("inferno_cache_evict", C.byref(a), C.c_void_p(ws.data_ptr()), ws.numel(), stream())


def evict_ref(k, v, scores, pos, lens, next_pos, scores_out, pos_out, *, budget, n_sink=0, n_recent=0, max_len=None):
    """The new (k, v, scores_out, pos_out, lens_out) on the CPU, row by row."""
    k, v, scores_out, pos_out = (x.cpu().clone() for x in (k, v, scores_out, pos_out))
    scores, pos, next_pos = scores.cpu(), pos.cpu(), next_pos.cpu()
    B, rows, H, _ = k.shape
    left = []
    for b in range(B):
        n = max(0, min(int(lens[b]), max_len or rows))
        now = min(n, budget)
        left.append(now)
        for h in range(H):
            def rank(j):
                s, at = float(scores[b, h, j]), int(pos[b, h, j])
                always = at < n_sink or at >= int(next_pos[b]) - n_recent
                return (not always, math.isnan(s), 0.0 if math.isnan(s) else -s, j)
            kept = sorted(sorted(range(n), key=rank)[:now]) if n > budget else list(range(n))
            inside = set(j for j in kept if j < now)
            behind = [j for j in kept if j >= now]
            source = [j if j in inside else None for j in range(now)]
            it = iter(behind)
            source = [next(it) if j is None else j for j in source]
            src = torch.tensor(source, dtype=torch.long)
            k[b, :now, h], v[b, :now, h] = k[b, src, h], v[b, src, h]
            scores_out[b, h, :now], pos_out[b, h, :now] = scores[b, h, src], pos[b, h, src]
    return k, v, scores_out, pos_out, torch.tensor(left, dtype=torch.int32)


__all__ = [n for n in dir() if not n.startswith("_")]
_ = lib
