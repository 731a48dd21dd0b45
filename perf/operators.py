"""Timed cases of the single-op entry points that a quantised transformer block is made of.

``op_gate_norm``        h' = a h + gate * post(y),  n = pre(h') * (1 + scale) + shift: what stands between two sub-layers of a block
``op_quantize_int8``    rows to 8-bit integers with one scale per token, and
``op_gemm_int8``        their product with 8-bit weights that have one scale per output channel, with the epilogues of ``op_gemm``
``op_rope_table``       cosines and sines of rotary positions on one or several axes, scaled for contexts beyond the trained one
``op_rope``             their application to query and key heads

``run`` computes a case in elementary torch operations, or with ``own`` through the engine's entry points, on the same inputs.  ``exact`` is the
definition in 64 bits.  Kinds of cases: "linear" (16-bit activations in, quantised per token, multiplied: what replaces one Linear), "norm", "entry" (a norm
that hands its rows to the product in 8 bits: the way into a block), "table" and "rope".
"""
import functools
import math

import numpy as np
import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPILOGUES = ("bias", "gelu", "silu", "resid")  # op_gemm's epilogues 0 .. 3
EPS = 1e-6


@functools.lru_cache(maxsize=None)
def _engine(dtype):
    """The handle that a program keeps: the smallest engine of that type."""
    from ecad_amd.engine import EcadEngine

    return EcadEngine(num_layers=1, num_heads=16, caption_channels=64, max_batch=1, max_tokens=64, max_text_tokens=8, dtype=TYPES[dtype])


# ---- cases ----------------------------------------------------------------------------------------------------------------------------------------------


def listed():
    return [
        # feed-forward of 28 blocks of width 1152 over 16 images of 256 tokens, doubled for guidance: up with GELU, down onto the gated residual
        dict(name="linear_ff1", kind="linear", dtype="fp16", m=8192, n=4608, k=1152, epi="gelu", batch=32),
        dict(name="linear_ff2", kind="linear", dtype="bf16", m=8192, n=1152, k=4608, epi="resid", batch=32),
        # text tokens of a prompt pair projected at odd widths: nothing is a whole tile, the last 16 bytes of a row are cut
        dict(name="linear_ragged", kind="linear", dtype="bf16", m=601, n=1111, k=4001, epi="silu", batch=1),
        # the modulation of all sub-layers from eight timestep embeddings: few rows, a whole weight matrix to read
        dict(name="linear_rows", kind="linear", dtype="fp16", m=8, n=6912, k=1152, epi="bias", batch=1),
        # between two sub-layers of that model: gated residual, LayerNorm, modulation
        dict(name="norm_block", kind="norm", dtype="fp16", m=8192, d=1152, post="none", pre="layer", batch=32, scale=1.0),
        # norms on both sides of a wide sub-layer, RMS, residual scaled as deep stacks do
        dict(name="norm_sandwich", kind="norm", dtype="bf16", m=16384, d=4096, post="rms", pre="rms", batch=4, scale=0.81),
        # one token per sequence at an odd width: latency
        dict(name="norm_step", kind="norm", dtype="bf16", m=5, d=1153, post="rms", pre="layer", batch=5, scale=1.0),
        # into a block: gated residual, norm, query/key/value projection of 8-bit rows
        dict(name="entry_qkv", kind="entry", dtype="bf16", m=4096, d=1152, n=3456, post="none", pre="layer", batch=16, scale=1.0),
        # image tokens behind text tokens, three axes, pairs side by side, heads inside the fused projection
        dict(name="rope_joint", kind="rope", dtype="bf16", b=2, s=4608, h=16, hk=16, d=128, rot=128, layout="interleaved", rows=4608, indexed=False),
        # one new token per sequence far into a long context, part of the head, pairs half a head apart, four query heads on a key head
        dict(name="rope_step", kind="rope", dtype="fp16", b=8, s=1, h=32, hk=8, d=72, rot=48, layout="half", rows=131072, indexed=True),
        # positions of a 128 x 128 latent on three axes, and of a long context scaled sixteen times
        dict(name="table_image", kind="table", s=16384, axes="16+56+56", theta=10000.0, scaling="none", factor=1.0, original=4096),
        dict(name="table_long", kind="table", s=131072, axes="128", theta=10000.0, scaling="yarn", factor=16.0, original=8192),
    ]


def _axes(case):
    return tuple(map(int, case["axes"].split("+")))


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "norm", "entry", "rope", "table"))
    dtype = rng.choice(tuple(TYPES))
    if kind == "linear":
        m, n, k = _spread(rng, 1, 8192), _spread(rng, 16, 8192), _spread(rng, 32, 8192)
        k = min(k, max(32, 8192 * 4608 * 1152 // (m * n)))
        return dict(kind=kind, dtype=dtype, m=m, n=n, k=k, epi=rng.choice(EPILOGUES), batch=rng.randint(1, min(m, 8)))
    if kind in ("norm", "entry"):
        m, d = _spread(rng, 1, 16384), _spread(rng, 64, 8192)
        d = min(d, 16384 * 4096 // m)
        case = dict(kind=kind, dtype=dtype, m=m, d=d, post=rng.choice(("none", "rms", "layer")), pre=rng.choice(("rms", "layer")), batch=rng.randint(1, min(m, 8)),
                    scale=rng.choice((1.0, round(rng.uniform(0.3, 2.0), 3))))
        if kind == "entry":
            case["m"] = m = min(m, 4096)
            case["n"] = _spread(rng, 16, max(16, min(8192, 8192 * 4608 * 1152 // (m * d))))
        return case
    if kind == "rope":
        d = 2 * rng.randint(4, 128)
        h, rows = _spread(rng, 1, 32), _spread(rng, 64, 131072)
        most = 2 * 4608 * 16 * 128 // (h * d)  # sequence positions that cost as much as the largest listed case
        s = _spread(rng, 1, min(8192, most))
        b = rng.randint(1, max(1, min(8, most // s)))
        rot = d if rng.random() < 0.5 else 2 * rng.randint(1, d // 2)
        indexed = rng.random() < 0.5
        return dict(kind=kind, dtype=dtype, b=b, s=s, h=h, hk=rng.randint(1, h), d=d, rot=rot, layout=rng.choice(("interleaved", "half")), rows=rows if indexed else s + rng.randint(0, 7),
                    indexed=indexed)
    axes = tuple(2 * rng.randint(1, 42) for _ in range(rng.randint(1, 3)))
    scaling = rng.choice(("none", "linear", "ntk", "yarn"))
    return dict(kind=kind, s=_spread(rng, 1, min(131072, 131072 * 128 // sum(axes))), axes="+".join(map(str, axes)), theta=rng.choice((10000.0, 500000.0)), scaling=scaling,
                factor=1.0 if scaling == "none" else round(rng.uniform(1.0, 16.0), 2), original=rng.choice((1024, 4096, 8192)))


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------------------------


def _weights(gen, n, k):
    """[n, k] weights as 8-bit integers with a scale per output channel, rows on 16 bytes: what a program keeps of a Linear."""
    w = torch.randn((n, k), generator=gen, device="cuda") * (0.5 + torch.rand((n, 1), generator=gen, device="cuda"))
    scale = w.abs().amax(1) / 127.0
    rows = torch.zeros((n, (k + 15) // 16 * 16), device="cuda", dtype=torch.int8)
    rows[:, :k] = torch.round(w / scale[:, None]).to(torch.int8)
    return rows[:, :k], scale / math.sqrt(k)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    st = {"case": case}
    if case["kind"] == "table":
        far = 1 if len(_axes(case)) > 1 else 8
        ids = torch.randint(0, far * case["s"], (case["s"], len(_axes(case))), generator=gen, device="cuda", dtype=torch.int32)
        return st | {"positions": ids}
    dt = TYPES[case["dtype"]]
    if case["kind"] == "rope":
        b, s, h, hk, d, rot = (case[x] for x in ("b", "s", "h", "hk", "d", "rot"))
        qkv = normal(b, s, (h + 2 * hk) * d).to(dt)  # q and k are columns of the fused projection
        place = torch.arange(case["rows"], device="cuda", dtype=torch.float64) + torch.randint(0, 1000, (1,), generator=gen, device="cuda")
        angle = place[:, None] * 10000.0 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / rot)
        st["table"] = torch.stack((angle.cos(), angle.sin()), -1).float()
        st["index"] = torch.randint(0, case["rows"], (b, s), generator=gen, device="cuda", dtype=torch.int32) if case["indexed"] else None
        st["q"] = qkv[:, :, : h * d].view(b, s, h, d)
        st["k"] = qkv[:, :, h * d : (h + hk) * d].view(b, s, hk, d)
        return st
    m, batch = case["m"], case["batch"]
    st["rows_per_batch"] = (m + batch - 1) // batch
    if case["kind"] == "linear":
        n, k = case["n"], case["k"]
        wide = torch.where(torch.rand((k,), generator=gen, device="cuda") < 0.01, 8.0, 1.0)  # a few channels are much larger, as behind a norm or a GELU
        st["x"] = (normal(m, k) * wide).to(dt)
        st["w"], st["w_scale"] = _weights(gen, n, k)
        st["bias"] = normal(n) * 0.1
        if case["epi"] == "resid":
            st["resid"] = normal(m, n).to(dt)
            st["gate_table"] = normal(n) * 0.3
            st["gate_mod"] = normal(batch, n).to(dt)
        return st
    d = case["d"]
    st["h"], st["y"] = (normal(m, d) * 2 + 0.25).to(dt), normal(m, d).to(dt)
    mod = (normal(batch, 3 * d) * 0.3).to(dt)  # gate, shift, scale side by side, as one projection of the timestep leaves them
    st["gate_mod"], st["mod_shift"], st["mod_scale"] = mod[:, :d], mod[:, d : 2 * d], mod[:, 2 * d :]
    st["gate_table"], st["table_shift"], st["table_scale"] = normal(d) * 0.3, normal(d) * 0.1, normal(d) * 0.1
    st["post_weight"] = 1 + 0.2 * normal(d) if case["post"] != "none" else None
    st["pre_weight"] = 1 + 0.2 * normal(d) if case["pre"] == "rms" else None
    if case["kind"] == "entry":
        st["w"], st["w_scale"] = _weights(gen, case["n"], d)
        st["bias"] = normal(case["n"]) * 0.1
    return st


# ---- the plain form -------------------------------------------------------------------------------------------------------------------------------------


def _frequencies(case):
    """Angle per unit of position of every pair (64 bits), its axis, and the factor on cosine and sine."""
    f, theta, axes = case["factor"], case["theta"], _axes(case)
    steep = [theta * f ** (a / (a - 2)) if case["scaling"] == "ntk" and a > 2 else theta for a in axes]
    freq = np.concatenate([t ** (-np.arange(a // 2) * 2.0 / a) for t, a in zip(steep, axes)])
    if case["scaling"] == "linear":
        freq = freq / f
    if case["scaling"] == "yarn":
        keep = np.clip((case["original"] * freq / (2 * np.pi) - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        freq = freq * (keep + (1 - keep) / f)
    return freq, np.repeat(np.arange(len(axes)), [a // 2 for a in axes]), 0.1 * math.log(f) + 1.0 if case["scaling"] == "yarn" else 1.0


def _plain_table(st):
    freq, axis, size = _frequencies(st["case"])
    angle = st["positions"][:, torch.from_numpy(axis).cuda()].double() * torch.from_numpy(freq).cuda()
    return torch.stack((angle.cos() * size, angle.sin() * size), -1).float()


def _plain_rotate(x, cos, sin, rot, layout):
    y = x.float()
    pairs = y[..., :rot].unflatten(-1, (rot // 2, 2) if layout == "interleaved" else (2, rot // 2))
    one, two = pairs.unbind(-1 if layout == "interleaved" else -2)
    turned = torch.stack((one * cos - two * sin, one * sin + two * cos), -1 if layout == "interleaved" else -2).flatten(-2)
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)


def _plain_rope(st):
    case = st["case"]
    at = st["table"][: case["s"]] if st["index"] is None else st["table"][st["index"].long()]
    cos, sin = at[..., None, :, 0], at[..., None, :, 1]
    return tuple(_plain_rotate(st[x], cos, sin, case["rot"], case["layout"]) for x in ("q", "k"))


def _plain_norm(x, kind, weight):
    if kind == "none":
        return x
    x = x - x.mean(1, keepdim=True) if kind == "layer" else x
    x = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    return x if weight is None else x * weight


def _per_row(st, table, mod):
    """table [d] + mod [sample, d] for every row."""
    m = st["case"]["m"]
    return st[table] + st[mod].float()[torch.arange(m, device="cuda") // st["rows_per_batch"]]


def _plain_gate_norm(st):
    case = st["case"]
    h = case["scale"] * st["h"].float() + _per_row(st, "gate_table", "gate_mod") * _plain_norm(st["y"].float(), case["post"], st["post_weight"])
    n = _plain_norm(h, case["pre"], st["pre_weight"]) * (1 + _per_row(st, "table_scale", "mod_scale")) + _per_row(st, "table_shift", "mod_shift")
    return h.to(st["h"].dtype), n.to(st["h"].dtype)


def _plain_quantize(x):
    scale = (x.double().abs().amax(1) / 127.0).float()  # the nearest fp32 value: torch divides fp32 by a number as a product with its reciprocal
    q = torch.round(x.double() / torch.where(scale > 0, scale, 1.0).double()[:, None])  # 64 bits: a value next to a border falls on its own side
    return q.float(), scale


def _plain_product(st, q, scale, epi):
    o = (q @ st["w"].float().t()) * scale[:, None] * st["w_scale"] + st["bias"]
    if epi == "gelu":
        o = 0.5 * o * (1 + torch.tanh(math.sqrt(2 / math.pi) * (o + 0.044715 * o * o * o)))
    if epi == "silu":
        o = o / (1 + torch.exp(-o))
    return o


def _plain_linear(st):
    dt = st["x"].dtype
    o = _plain_product(st, *_plain_quantize(st["x"]), st["case"]["epi"]).to(dt)
    if st["case"]["epi"] != "resid":
        return o
    return o, (st["resid"].float() + _per_row(st, "gate_table", "gate_mod") * o.float()).to(dt)  # what is cached is what the residual takes


def _plain_entry(st):
    h, n = _plain_gate_norm(st)
    return h, _plain_product(st, *_plain_quantize(n), "bias").to(h.dtype)


# ---- the engine's entry points --------------------------------------------------------------------------------------------------------------------------


def _own_linear(st):
    case, eng = st["case"], _engine(st["case"]["dtype"])
    q, scale = eng.op_quantize_int8(st["x"])
    epi = EPILOGUES.index(case["epi"])
    if case["epi"] != "resid":
        return eng.op_gemm_int8(epi, q, scale, st["w"], st["w_scale"], st["bias"])
    out, resid = torch.empty_like(st["resid"]), torch.empty_like(st["resid"])  # the updated residual apart, so that the next pass starts from the same one
    eng.op_gemm_int8(epi, q, scale, st["w"], st["w_scale"], st["bias"], resid=st["resid"], gate_table=st["gate_table"], gate_mod=st["gate_mod"],
                     rows_per_batch=st["rows_per_batch"], out=out, resid_out=resid)
    return out, resid


def _own_gate_norm(st, quantize=False):
    case = st["case"]
    return _engine(case["dtype"]).op_gate_norm(
        st["h"], st["y"], pre=case["pre"], post=case["post"], pre_weight=st["pre_weight"], post_weight=st["post_weight"], gate_table=st["gate_table"], gate_mod=st["gate_mod"],
        table_shift=st["table_shift"], table_scale=st["table_scale"], mod_shift=st["mod_shift"], mod_scale=st["mod_scale"], rows_per_batch=st["rows_per_batch"],
        resid_scale=case["scale"], eps=EPS, quantize=quantize)


def _own_entry(st):
    h, (q, scale) = _own_gate_norm(st, quantize=True)
    return h, _engine(st["case"]["dtype"]).op_gemm_int8(0, q, scale, st["w"], st["w_scale"], st["bias"])


def _own_rope(st):
    case = st["case"]
    return _engine(case["dtype"]).op_rope(st["q"], st["k"], st["table"], layout=case["layout"], index=st["index"])


def _own_table(st):
    case = st["case"]
    return _engine("fp16").op_rope_table(st["positions"], _axes(case), theta=case["theta"], scaling=case["scaling"], factor=case["factor"], original_length=case["original"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"linear": _own_linear, "norm": _own_gate_norm, "entry": _own_entry, "rope": _own_rope, "table": _own_table}[kind](state)
    return {"linear": _plain_linear, "norm": _plain_gate_norm, "entry": _plain_entry, "rope": _plain_rope, "table": _plain_table}[kind](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "table":
        pairs = sum(_axes(case)) // 2
        return {"bytes": case["s"] * (4 * len(_axes(case)) + 8 * pairs), "flops": 3 * case["s"] * pairs}
    if case["kind"] == "rope":
        values = case["b"] * case["s"] * (case["h"] + case["hk"])
        rows = case["b"] * case["s"] if case["indexed"] else case["s"]
        return {"bytes": 4 * values * case["d"] + 4 * min(rows, case["rows"]) * case["rot"] + (4 * rows if case["indexed"] else 0), "flops": 3 * values * case["rot"]}
    m = case["m"]
    if case["kind"] == "linear":
        n, k = case["n"], case["k"]
        resid = 4 * m * n + 2 * case["batch"] * n + 4 * n if case["epi"] == "resid" else 0
        return {"bytes": 2 * m * k + n * k + 2 * m * n + 8 * n + resid, "flops": 2 * m * n * k}
    d = case["d"]
    norm = 6 * m * d + 6 * case["batch"] * d + 12 * d
    if case["kind"] == "norm":
        return {"bytes": norm + 2 * m * d, "flops": 16 * m * d}
    return {"bytes": norm + case["n"] * d + 2 * m * case["n"] + 8 * case["n"], "flops": 2 * m * case["n"] * d + 16 * m * d}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------------------------------------


def _wide(t):
    return None if t is None else t.to(torch.float64)


def _exact_statistics_norm(x, kind, weight):
    if kind == "none":
        return x
    centre = x.sum(1, keepdim=True) / x.shape[1] if kind == "layer" else torch.zeros_like(x[:, :1])
    spread = ((x - centre) ** 2).sum(1, keepdim=True) / x.shape[1]
    x = (x - centre) / torch.sqrt(spread + EPS)
    return x if weight is None else x * _wide(weight)


def _exact_gate_norm(st):
    case = st["case"]
    sample = torch.div(torch.arange(case["m"], device="cuda"), st["rows_per_batch"], rounding_mode="floor")
    both = lambda table, mod: _wide(st[table])[None, :] + _wide(st[mod]).index_select(0, sample)  # noqa: E731
    h = _wide(st["h"]) * case["scale"] + _exact_statistics_norm(_wide(st["y"]), case["post"], st["post_weight"]) * both("gate_table", "gate_mod")
    n = _exact_statistics_norm(h, case["pre"], st["pre_weight"])
    return h, n + n * both("table_scale", "mod_scale") + both("table_shift", "mod_shift")


def _exact_product(st, x, epi):
    """The rows x, values of the storage type, in steps of the 32-bit scale."""
    largest = x.abs().max(1, keepdim=True).values
    step = (largest / 127.0).float().double()
    whole = torch.where(step > 0, x / step.clamp_min(1e-300), torch.zeros_like(x)).round()
    o = (whole * step) @ (_wide(st["w"]) * _wide(st["w_scale"])[:, None]).T + _wide(st["bias"])
    if epi == "gelu":
        return o / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (o + 0.044715 * o**3)))
    return o * torch.sigmoid(o) if epi == "silu" else o


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "table":
        place, f, columns = st["positions"].cpu().numpy().astype(np.float64), case["factor"], []
        size = 1 + math.log(f) / 10 if case["scaling"] == "yarn" else 1.0
        for axis, width in enumerate(_axes(case)):
            for j in range(width // 2):
                turns = case["theta"] ** (-2 * j / width)  # radians per unit of position
                if case["scaling"] == "linear":
                    turns /= f
                elif case["scaling"] == "ntk" and width > 2:
                    turns *= f ** (-2 * j / (width - 2))
                elif case["scaling"] == "yarn":  # pairs that turn 32 times within the original length stay, those that turn less than once are stretched
                    whole = min(1.0, max(0.0, (case["original"] * turns / (2 * math.pi) - 1) / 31))
                    turns = turns * whole + turns / f * (1 - whole)
                columns.append(np.stack((size * np.cos(place[:, axis] * turns), size * np.sin(place[:, axis] * turns)), -1))
        return torch.from_numpy(np.stack(columns, 1))
    if case["kind"] == "rope":
        rot, side = case["rot"], case["layout"] == "interleaved"
        rows = st["index"].long() if st["index"] is not None else torch.arange(case["s"], device="cuda").expand(case["b"], case["s"])
        turn = torch.complex(*_wide(st["table"])[rows].unbind(-1))[:, :, None, :]
        outs = []
        for x in (st["q"], st["k"]):
            x = _wide(x)
            z = torch.complex(x[..., 0:rot:2].contiguous(), x[..., 1:rot:2].contiguous()) if side else torch.complex(x[..., : rot // 2].contiguous(), x[..., rot // 2 : rot].contiguous())
            z = z * turn
            y = x.clone()
            if side:
                y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
            else:
                y[..., : rot // 2], y[..., rot // 2 : rot] = z.real, z.imag
            outs.append(y)
        return tuple(outs)
    if case["kind"] == "linear":
        o = _exact_product(st, _wide(st["x"]), case["epi"])
        if case["epi"] != "resid":
            return o
        sample = torch.arange(case["m"], device="cuda") // st["rows_per_batch"]
        return o, _wide(st["resid"]) + (_wide(st["gate_table"]) + _wide(st["gate_mod"])[sample]) * _wide(o.to(st["resid"].dtype))
    h, n = _exact_gate_norm(st)
    if case["kind"] == "norm":
        return h, n
    return h, _exact_product(st, _wide(n.to(st["h"].dtype)), "bias")
