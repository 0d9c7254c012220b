"""Cases of the long-context serving operators: rotary positions with the
cache append, attention over a shared prefix and per-sequence caches (with the
attention weight that each cached row gathers), and eviction from a cache by
that weight.

``own`` false computes them in plain torch operations; true calls
libinferno_b200.so.  Layouts are the engine's: a cache slice is
[rows][n_kv_heads][head_dim], a token row of q is [n_heads][head_dim].
"""
import ctypes
import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parent.parent / "inferno.jl_b200")
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}          # ggml type ids


def listed():
    return [
        # one decode step of 8 sequences: q rotated, k rotated and v copied into the caches at each sequence's row
        _rope("rope decode 8 f32 append", "f32", 8, 16, 4, 256, 64, append=True, max_pos=32768, theta=1e7),
        # a whole prompt after its fused q/k/v product, a quarter of each head rotated
        _rope("rope prompt 2048 f32", "f32", 2048, 16, 4, 256, 64, max_pos=2048, theta=1e7),
        # long prompts beyond the trained context: interleaved pairs, scaled by parts, an odd number of tokens
        _rope("rope long 16383 bf16 yarn", "bf16", 16383, 32, 8, 128, 128, layout=1, scaling=2, factor=8.0,
              max_pos=262144, theta=1e4, append=True),
        # four short chats on one system prompt: the smallest batched step
        _attn("prefix 500 x4 f32", "f32", 4, 1, 8, 2, 256, prefix=500, max_len=12),
        # eight sequences behind one 2048-token prompt, 256 steps of their own
        _attn("prefix 2048 x8 f32", "f32", 8, 1, 16, 4, 256, prefix=2048, max_len=256),
        # 64 samples of one prompt
        _attn("prefix 4096 x64 bf16", "bf16", 64, 1, 16, 2, 256, prefix=4096, max_len=128),
        # a long document asked 32 questions; lengths that end inside tiles
        _attn("prefix 32001 x32 bf16", "bf16", 32, 1, 32, 8, 128, prefix=32001, max_len=777),
        # draft tokens of five sequences verified together
        _attn("prefix 1000 x5 t4 f16", "f16", 5, 4, 12, 4, 64, prefix=1000, max_len=333),
        # one sequence in a short cache, rows' weight gathered for eviction
        _attn("weights 500 x1 f32", "f32", 1, 1, 8, 2, 256, max_len=500, weights=True),
        # sixteen sequences at up to 16k rows each
        _attn("weights 16384 x16 bf16", "bf16", 16, 1, 32, 8, 128, max_len=16384, weights=True),
        # the step after each block of 64 tokens: a full budget plus the block
        _evict("evict 4160 to 4096 f32", "f32", 8, 4, 256, 4160, 4096, 4, 256),
        # a prompt cut to its budget
        _evict("evict 32768 to 4096 bf16", "bf16", 4, 8, 128, 32768, 4096, 4, 512),
    ]


def _rope(name, dtype, tokens, heads, kv, dim, rope_dim, layout=0, scaling=0, factor=1.0, max_pos=4096, theta=1e4,
          append=False):
    return dict(name=name, op="rope", dtype=dtype, tokens=tokens, heads=heads, kv=kv, dim=dim, rope_dim=rope_dim,
                layout=layout, scaling=scaling, factor=factor, max_pos=max_pos, theta=theta, append=append)


def _attn(name, dtype, batch, tokens, heads, kv, dim, prefix=0, max_len=0, weights=False):
    return dict(name=name, op="attention", dtype=dtype, batch=batch, tokens=tokens, heads=heads, kv=kv, dim=dim,
                prefix=prefix, max_len=max_len, weights=weights)


def _evict(name, dtype, batch, kv, dim, max_len, budget, sink, recent):
    return dict(name=name, op="evict", dtype=dtype, batch=batch, kv=kv, dim=dim, max_len=max_len, budget=budget,
                sink=sink, recent=recent)


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["f32", "f16", "bf16"])
    kv, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8]), rng.choice([64, 128, 256])
    kind = rng.choice(["rope", "prefix", "weights", "evict"])
    size = 4 if dtype == "f32" else 2
    if kind == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        tokens = max(1, min(_between(rng, 1, 16383), int(3e8 / ((group + 2) * kv * dim * size))))
        c = _rope("", dtype, tokens, kv * group, kv, dim, rng.choice([dim, dim // 2, dim // 4]), rng.choice([0, 1]),
                  rng.choice([0, 1, 2]), rng.choice([2.0, 4.0, 16.0]), _between(rng, 512, 1 << 20),
                  rng.choice([1e4, 5e5, 1e7]), rng.choice([True, False]))
    elif kind == "prefix":
        batch, tokens = _between(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 8])
        prefix, max_len = _between(rng, 16, 32768), _between(rng, tokens, 2048)
        per_key = batch * tokens * kv * group * dim * (4 if dtype == "f32" else 1)   # products of a prefix row
        prefix = max(1, min(prefix, int(2.5e9 / per_key)))
        max_len = max(tokens, min(max_len, int(4e8 / (batch * kv * dim * size))))
        c = _attn("", dtype, batch, tokens, kv * group, kv, dim, prefix, max_len)
    elif kind == "weights":
        batch, tokens = _between(rng, 1, 32), rng.choice([1, 1, 1, 2, 4])
        max_len = max(tokens, min(_between(rng, 16, 65536), int(4e8 / (batch * kv * dim * size))))
        c = _attn("", dtype, batch, tokens, kv * group, kv, dim, 0, max_len, True)
    else:
        batch = _between(rng, 1, 16)
        max_len = max(16, min(_between(rng, 16, 65536), int(4e8 / (batch * kv * dim * size))))
        budget = max(8, int(max_len * rng.uniform(0.1, 0.99)))
        c = _evict("", dtype, batch, kv, dim, max_len, budget, rng.choice([0, 1, 4]), rng.randint(0, budget // 2))
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"case": case, **_PREPARE[case["op"]](case, gen)}


def _randn(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _randint(gen, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=gen, device="cuda", dtype=torch.int32)


def _rope_inputs(c, gen):
    dt, n, d = _TYPES[c["dtype"]], c["tokens"], c["dim"]
    qkv = _randn(gen, dt, n, (c["heads"] + 2 * c["kv"]) * d)      # the fused product's rows
    q, k, v = qkv.split([c["heads"] * d, c["kv"] * d, c["kv"] * d], dim=1)
    s = dict(q=q, k=k, v=v, q_out=torch.empty(n, c["heads"] * d, dtype=dt, device="cuda"),
             positions=_randint(gen, 0, c["max_pos"], n),
             factors=torch.rand(c["rope_dim"] // 2, generator=gen, device="cuda") + 0.5 if c["scaling"] == 1 else None)
    if c["append"]:                                               # caches with room for the rows of other steps
        rows = n + 8 + n // 4
        s["slots"] = torch.randperm(rows, generator=gen, device="cuda")[:n].to(torch.int32)
        s["k_out"], s["v_out"] = _randn(gen, dt, rows, c["kv"] * d), _randn(gen, dt, rows, c["kv"] * d)
    else:
        s["k_out"] = torch.empty(n, c["kv"] * d, dtype=dt, device="cuda")
    return s


def _attn_inputs(c, gen):
    dt, B, T, H, d = _TYPES[c["dtype"]], c["batch"], c["tokens"], c["kv"], c["dim"]
    s = dict(q=_randn(gen, dt, B, T, c["heads"], d) * 2, out=torch.empty(B, T, c["heads"], d, dtype=dt, device="cuda"),
             k=_randn(gen, dt, B, c["max_len"], H, d), v=_randn(gen, dt, B, c["max_len"], H, d),
             lens=_randint(gen, min(c["max_len"], max(T, c["max_len"] // 2)), c["max_len"] + 1, B))
    if c["prefix"]:
        s["pk"], s["pv"] = _randn(gen, dt, c["prefix"], H, d), _randn(gen, dt, c["prefix"], H, d)
    if c["weights"]:
        s["scores"] = torch.rand(B, H, c["max_len"], generator=gen, device="cuda")
    return s


def _evict_inputs(c, gen):
    dt, B, H, L = _TYPES[c["dtype"]], c["batch"], c["kv"], c["max_len"]
    # gathered weights have a long tail: a few rows hold most
    scores = torch.rand(B, H, L, generator=gen, device="cuda").clamp_min(1e-7).pow(-0.7) - 1
    order = torch.rand(B, H, L, generator=gen, device="cuda").argsort(-1).to(torch.int32)   # earlier evictions moved rows
    return dict(k=_randn(gen, dt, B, L, H, c["dim"]), v=_randn(gen, dt, B, L, H, c["dim"]), scores=scores, pos=order,
                lens=torch.full((B,), L, dtype=torch.int32, device="cuda"),
                next_pos=torch.full((B,), L, dtype=torch.int32, device="cuda"),
                scores_out=torch.zeros(B, H, L, device="cuda"),
                pos_out=torch.zeros(B, H, L, dtype=torch.int32, device="cuda"),
                lens_out=torch.zeros(B, dtype=torch.int32, device="cuda"))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    return _OWN[op](state) if own else _PLAIN[op](state)


def _frequencies(c, factors, kind):
    """Angle per position of each rotated pair, and the factor of cos and sin."""
    half = c["rope_dim"] // 2
    i = torch.arange(half, device="cuda", dtype=kind)
    freq = c["theta"] ** (-2.0 * i / c["rope_dim"])
    if factors is not None:
        freq = freq / factors.to(kind)
    if c["scaling"] == 0:
        return freq, 1.0
    if c["scaling"] == 1:
        return freq / c["factor"], 1.0
    # by parts: pairs that turn often keep their angle, pairs that turn rarely are interpolated
    at = [c["rope_dim"] * math.log(_TRAINED / (turns * 2 * math.pi)) / (2 * math.log(c["theta"])) for turns in (32.0, 1.0)]
    low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), c["rope_dim"] - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return freq / c["factor"] * ramp + freq * (1 - ramp), 0.1 * math.log(c["factor"]) + 1.0


_TRAINED = 4096     # positions of the context before scaling


def _rotate(c, x, cos, sin):
    """x [tokens][heads][dim], cos and sin [tokens][1][pairs]."""
    r = c["rope_dim"]
    if c["layout"] == 0:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _rope_plain(s):
    c = s["case"]
    freq, m = _frequencies(c, s["factors"], torch.float64)
    angle = s["positions"].double()[:, None, None] * freq
    cos, sin = (angle.cos() * m).float(), (angle.sin() * m).float()
    q = _rotate(c, s["q"].float().unflatten(1, (c["heads"], c["dim"])), cos, sin)
    k = _rotate(c, s["k"].float().unflatten(1, (c["kv"], c["dim"])), cos, sin)
    s["q_out"].copy_(q.flatten(1))
    if not c["append"]:
        s["k_out"].copy_(k.flatten(1))
        return s["q_out"], s["k_out"]
    s["k_out"][s["slots"]] = k.flatten(1).to(s["k_out"].dtype)
    s["v_out"][s["slots"]] = s["v"]
    return s["q_out"], s["k_out"], s["v_out"]


def _attn_plain(s):
    c = s["case"]
    B, T, H, d, L, P = c["batch"], c["tokens"], c["kv"], c["dim"], c["max_len"], c["prefix"]
    q = s["q"].float().view(B, T, H, -1, d) / math.sqrt(d)
    own_s = torch.einsum("bthgd,blhd->bhtgl", q, s["k"].float())
    # token t of T sees the rows up to its own: the last T rows are those of the T tokens
    seen = s["lens"][:, None] - (T - 1) + torch.arange(T, device="cuda")
    mask = torch.arange(L, device="cuda") < seen[:, :, None]
    own_s = own_s.masked_fill(~mask[:, None, :, None, :], -math.inf)
    both = own_s
    if P:
        both = torch.cat([torch.einsum("bthgd,phd->bhtgp", q, s["pk"].float()), own_s], -1)
    top = both.amax(-1, keepdim=True)
    e = torch.exp(both - torch.where(top == -math.inf, 0.0, top))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    live = torch.arange(L, device="cuda") < s["lens"][:, None]
    o = torch.einsum("bhtgl,blhd->bthgd", p[..., P:], s["v"].float().masked_fill(~live[:, :, None, None], 0.0))
    if P:
        o = o + torch.einsum("bhtgp,phd->bthgd", p[..., :P], s["pv"].float())
    s["out"].copy_(o.reshape(B, T, -1, d))
    if c["weights"]:
        s["scores"] += p[..., P:].sum((2, 3))
        return s["out"], s["scores"]
    return s["out"]


def _evict_plain(s):
    c = s["case"]
    slot = torch.arange(c["max_len"], device="cuda")
    lens = s["lens"][:, None, None]
    live = (slot < lens).expand_as(s["scores"])
    kept_always = (s["pos"] < c["sink"]) | (s["pos"] >= s["next_pos"][:, None, None] - c["recent"])
    key = s["scores"].masked_fill(kept_always, math.inf).masked_fill(~live, -math.inf)
    first = key.sort(dim=-1, descending=True, stable=True).indices[..., :c["budget"]]
    keep = torch.zeros_like(live).scatter_(-1, first, True)
    keep = torch.where(lens > c["budget"], keep, live)
    # the rows that are kept behind the budget fill the holes before it, both in rising order
    hb, hh, to = (~keep & live & (slot < c["budget"])).nonzero(as_tuple=True)
    _, _, fro = (keep & (slot >= c["budget"])).nonzero(as_tuple=True)
    s["k"][hb, to, hh] = s["k"][hb, fro, hh]
    s["v"][hb, to, hh] = s["v"][hb, fro, hh]
    left = torch.minimum(s["lens"], torch.full_like(s["lens"], c["budget"]))
    stays = slot < left[:, None, None]
    for out, x in ((s["scores_out"], s["scores"]), (s["pos_out"], s["pos"])):
        out.copy_(torch.where(stays, x, out))
        out[hb, hh, to] = x[hb, hh, fro]
    s["lens_out"].copy_(left)
    return s["k"], s["v"], s["scores_out"], s["pos_out"], s["lens_out"]


def _library():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from inferno_b200 import _lib
    return _lib


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _rope_own(s):
    c, L = s["case"], _library()
    out = [s["q_out"], s["k_out"]]
    a = L.InfernoRope(type=_TYPE_IDS[c["dtype"]], n_tokens=c["tokens"], n_heads=c["heads"], n_kv_heads=c["kv"],
                      head_dim=c["dim"], rope_dim=c["rope_dim"], layout=c["layout"], scaling=c["scaling"],
                      theta=c["theta"], factor=c["factor"], orig_ctx=_TRAINED, positions=s["positions"].data_ptr(),
                      q=s["q"].data_ptr(), k=s["k"].data_ptr(), q_stride=s["q"].stride(0), k_stride=s["k"].stride(0),
                      q_out=s["q_out"].data_ptr(), k_out=s["k_out"].data_ptr(), q_out_stride=s["q_out"].stride(0),
                      k_out_stride=s["k_out"].stride(0))
    if s["factors"] is not None:
        a.freq_factors = s["factors"].data_ptr()
    if c["append"]:
        a.slots, a.n_rows = s["slots"].data_ptr(), s["k_out"].shape[0]
        a.v, a.v_stride = s["v"].data_ptr(), s["v"].stride(0)
        a.v_out, a.v_out_stride = s["v_out"].data_ptr(), s["v_out"].stride(0)
        out.append(s["v_out"])
    L.call("inferno_rope", ctypes.byref(a), _stream())
    return tuple(out)


def _attn_own(s):
    c, L = s["case"], _library()
    a = L.InfernoAttention(type=_TYPE_IDS[c["dtype"]], batch=c["batch"], n_tokens=c["tokens"], n_heads=c["heads"],
                           n_kv_heads=c["kv"], head_dim=c["dim"], prefix_len=c["prefix"], max_len=c["max_len"],
                           q_stride=s["q"].stride(1), out_stride=s["out"].stride(1), seq_stride=s["k"].stride(0),
                           q=s["q"].data_ptr(), k_cache=s["k"].data_ptr(), v_cache=s["v"].data_ptr(),
                           lens=s["lens"].data_ptr(), out=s["out"].data_ptr())
    if c["prefix"]:
        a.prefix_k, a.prefix_v = s["pk"].data_ptr(), s["pv"].data_ptr()
    if c["weights"]:
        a.scores, a.score_stride = s["scores"].data_ptr(), s["scores"].stride(1)
    n = L.call("inferno_attention_cached_workspace", ctypes.byref(a))
    work_area = torch.empty(n, dtype=torch.uint8, device="cuda")
    L.call("inferno_attention_cached", ctypes.byref(a), ctypes.c_void_p(work_area.data_ptr()), n, _stream())
    return (s["out"], s["scores"]) if c["weights"] else s["out"]


def _evict_own(s):
    c, L = s["case"], _library()
    a = L.InfernoEvict(type=_TYPE_IDS[c["dtype"]], batch=c["batch"], n_kv_heads=c["kv"], head_dim=c["dim"],
                       max_len=c["max_len"], budget=c["budget"], n_sink=c["sink"], n_recent=c["recent"],
                       seq_stride=s["k"].stride(0), score_stride=s["scores"].stride(1), k_cache=s["k"].data_ptr(),
                       v_cache=s["v"].data_ptr(), scores=s["scores"].data_ptr(), slot_pos=s["pos"].data_ptr(),
                       lens=s["lens"].data_ptr(), next_pos=s["next_pos"].data_ptr(),
                       scores_out=s["scores_out"].data_ptr(), slot_pos_out=s["pos_out"].data_ptr(),
                       lens_out=s["lens_out"].data_ptr())
    n = L.call("inferno_cache_evict_workspace", ctypes.byref(a))
    work_area = torch.empty(n, dtype=torch.uint8, device="cuda")
    L.call("inferno_cache_evict", ctypes.byref(a), ctypes.c_void_p(work_area.data_ptr()), n, _stream())
    return s["k"], s["v"], s["scores_out"], s["pos_out"], s["lens_out"]


_PREPARE = {"rope": _rope_inputs, "attention": _attn_inputs, "evict": _evict_inputs}
_PLAIN = {"rope": _rope_plain, "attention": _attn_plain, "evict": _evict_plain}
_OWN = {"rope": _rope_own, "attention": _attn_own, "evict": _evict_own}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c, size = case, 4 if case["dtype"] == "f32" else 2
    if c["op"] == "rope":
        values = c["tokens"] * (c["heads"] + (2 if c["append"] else 1) * c["kv"]) * c["dim"]
        turned = c["tokens"] * (c["heads"] + c["kv"]) * c["rope_dim"]
        return {"bytes": 2 * values * size + c["tokens"] * (8 if c["append"] else 4), "flops": 3 * turned}
    if c["op"] == "attention":
        # own lengths are spread evenly over [max(tokens, max_len / 2), max_len]
        mean = (min(c["max_len"], max(c["tokens"], c["max_len"] // 2)) + c["max_len"]) / 2
        rows = c["prefix"] + c["batch"] * mean
        q = c["batch"] * c["tokens"] * c["heads"] * c["dim"]
        weights = 8 * c["batch"] * c["kv"] * mean if c["weights"] else 0
        return {"bytes": 2 * q * size + 2 * rows * c["kv"] * c["dim"] * size + weights + 4 * c["batch"],
                "flops": 4 * q * (c["prefix"] + mean)}
    # the rows that move: kept ones behind the budget, in expectation
    heads, behind = c["batch"] * c["kv"], c["max_len"] - c["budget"]
    moved = heads * behind * c["budget"] / c["max_len"]
    return {"bytes": heads * 8 * (c["max_len"] + c["budget"]) + 4 * moved * c["dim"] * size + 12 * c["batch"],
            "flops": heads * c["max_len"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    return _EXACT[case["op"]](case, prepare(case, seed))


def _rope_exact(c, s):
    n, half = c["tokens"], c["rope_dim"] // 2
    base = torch.tensor(float(c["theta"]), dtype=torch.float64, device="cuda")
    pair = torch.arange(half, dtype=torch.float64, device="cuda")
    wave = torch.exp(-torch.log(base) * (2 * pair / c["rope_dim"]))
    if s["factors"] is not None:
        wave = wave / s["factors"].double()
    gain = 1.0
    if c["scaling"] == 1:
        wave = wave / c["factor"]
    elif c["scaling"] == 2:
        bound = []
        for turns in (32, 1):      # the pair that makes so many turns over the trained context
            bound.append(c["rope_dim"] / 2 * math.log(_TRAINED / (2 * math.pi * turns)) / math.log(c["theta"]))
        first, last = max(0, math.floor(bound[0])), min(c["rope_dim"] - 1, math.ceil(bound[1]))
        share = torch.clamp((pair - first) / max(last - first, 0.001), 0.0, 1.0)
        wave = wave * (1 - share + share / c["factor"])
        gain = 1.0 + 0.1 * math.log(c["factor"])
    turn = torch.polar(torch.full((n, half), gain, dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * wave)
    place = torch.arange(c["rope_dim"], device="cuda").view(2, half) if c["layout"] == 0 \
        else torch.arange(c["rope_dim"], device="cuda").view(half, 2).t()
    done = []
    for x, heads in ((s["q"], c["heads"]), (s["k"], c["kv"])):
        y = x.double().reshape(n, heads, c["dim"]).clone()
        z = torch.complex(y[..., place[0]], y[..., place[1]]) * turn[:, None, :]
        y[..., place[0]], y[..., place[1]] = z.real, z.imag
        done.append(y.reshape(n, -1))
    if not c["append"]:
        return tuple(done)
    k, v = s["k_out"].double(), s["v_out"].double()
    k.index_copy_(0, s["slots"].long(), done[1])
    v.index_copy_(0, s["slots"].long(), s["v"].double())
    return done[0], k, v


def _attn_exact(c, s):
    T, H, d = c["tokens"], c["kv"], c["dim"]
    group = c["heads"] // H
    out = torch.zeros(c["batch"], T, c["heads"], d, dtype=torch.float64, device="cuda")
    gathered = s["scores"].double() if c["weights"] else None
    for b, n in enumerate(s["lens"].tolist()):
        for h in range(H):
            keys, values = s["k"][b, :n, h].double(), s["v"][b, :n, h].double()
            if c["prefix"]:
                keys = torch.cat([s["pk"][:, h].double(), keys])
                values = torch.cat([s["pv"][:, h].double(), values])
            for t in range(T):
                seen = c["prefix"] + max(0, n - (T - 1) + t)
                if not seen:
                    continue
                logits = s["q"][b, t, h * group:(h + 1) * group].double() @ keys[:seen].t() * d ** -0.5
                p = torch.softmax(logits, -1)
                out[b, t, h * group:(h + 1) * group] = p @ values[:seen]
                if c["weights"]:
                    gathered[b, h, :seen - c["prefix"]] += p[:, c["prefix"]:].sum(0)
    return (out, gathered) if c["weights"] else out


def _evict_exact(c, s):
    k, v = s["k"].double(), s["v"].double()
    scores, pos = torch.zeros_like(s["scores"], dtype=torch.float64), torch.zeros_like(s["pos"])
    left = []
    for b, n in enumerate(s["lens"].tolist()):
        now = min(n, c["budget"])
        left.append(now)
        for h in range(c["kv"]):
            where, weight = s["pos"][b, h, :n].cpu(), s["scores"][b, h, :n].cpu().double()
            safe = (where < c["sink"]) | (where >= int(s["next_pos"][b]) - c["recent"])
            kept = torch.zeros(n, dtype=torch.bool)
            kept[safe] = True
            others = (~safe).nonzero().flatten()
            ranked = others[torch.sort(weight[others], descending=True, stable=True).indices]
            kept[ranked[:max(0, now - int(safe.sum()))]] = True
            source = torch.arange(now)
            source[~kept[:now]] = now + kept[now:].nonzero().flatten()
            at = source.cuda()
            k[b, :now, h], v[b, :now, h] = k[b, at, h], v[b, at, h]
            scores[b, h, :now] = weight[source].cuda()
            pos[b, h, :now] = where[source].to(torch.int32).cuda()
    return k, v, scores, pos, torch.tensor(left, dtype=torch.int32, device="cuda")


_EXACT = {"rope": _rope_exact, "attention": _attn_exact, "evict": _evict_exact}
