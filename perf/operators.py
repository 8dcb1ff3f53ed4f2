"""The operators of a decode step around the 4-bit weight products, as cases to be measured.

  matvec   Y = act(alpha * X dequant(W)^T + beta * C + bias), 1 to 16 rows of X, W in 4 bits with one scale (and
           optionally one zero point) per group of 32, 64 or 128 along K
  rotary   rotary positions on the heads of a projection's result, forward and backward
  logits   penalties for repeated tokens, biases and grammar masks on the rows of the head product

`own` False: the plain forms below, elementary torch operations in 32 bits.  `own` True: the calls a user makes of
the framework (sm120_gemm_b200).
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TYPE_IDS = {"bf16": 0, "f16": 1, "f32": 2}
ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


# ------------------------------------------------------------------------------------------------------------- cases
def _matvec(m, n, k, group, dtype, zeros, act="none", bias=False, residual=False, **name):
    return dict(name, op="matvec", m=m, n=n, k=k, group=group, dtype=dtype, zeros=zeros, act=act, bias=bias, residual=residual)


def _rotary(tokens, heads, extra, dim, rot, layout, dtype, scaling, far, backward=False, padded=False, **name):
    return dict(name, op="rotary", tokens=tokens, heads=heads, extra=extra, dim=dim, rot=rot, layout=layout, dtype=dtype, scaling=scaling, far=far,
                backward=backward, padded=padded)


def _logits(rows, vocab, history, dtype, out, biases, mask, penalties=True, **name):
    return dict(name, op="logits", rows=rows, vocab=vocab, history=history, dtype=dtype, out=out, biases=biases, mask=mask, penalties=penalties)


def listed():
    return [
        # one token through a square projection: the smallest product of a decode step, where latency counts
        _matvec(1, 4096, 4096, 128, "bf16", False, name="matvec_square_1"),
        # one token through the wide projection of the benchmark's decode shape
        _matvec(1, 28672, 8192, 128, "bf16", False, name="matvec_wide_1"),
        # sixteen sequences decoded together through the same weights, with zero points
        _matvec(16, 28672, 8192, 128, "bf16", True, name="matvec_wide_16"),
        # the long reduction of the second decode shape, fine groups, half precision, added to the residual stream
        _matvec(2, 4096, 14336, 32, "f16", True, residual=True, name="matvec_long_2"),
        # odd sizes: neither the rows nor K fill a tile; bias and activation fused
        _matvec(5, 5003, 6304, 32, "bf16", False, act="silu", bias=True, name="matvec_odd_5"),
        # the head product over a large vocabulary for four sequences: the largest weight of a decode step
        _matvec(4, 131072, 4096, 64, "bf16", False, name="matvec_head_4"),
        # queries and keys of 16 decoded tokens inside the fused QKV result, far into a long context
        _rotary(16, 40, 8, 128, 128, "half", "bf16", "ramp", 1 << 20, name="rotary_decode"),
        # a prompt of 8192 tokens
        _rotary(8192, 40, 8, 128, 128, "half", "bf16", "none", 8192, name="rotary_prompt"),
        # training: the gradient through interleaved pairs on part of the head, padded, an odd number of tokens
        _rotary(6001, 24, 0, 96, 64, "interleaved", "f16", "linear", 32768, backward=True, padded=True, name="rotary_gradient"),
        # one sequence: penalties and a few biases, a short history and an odd vocabulary
        _logits(1, 32001, 300, "bf16", "f32", 12, False, name="logits_one"),
        # a batch of 64 sequences under grammar masks
        _logits(64, 131072, 4096, "bf16", "f32", 64, True, name="logits_batch"),
        # few sequences with long histories, odd vocabulary, 32-bit logits
        _logits(8, 100003, 60000, "f32", "f32", 300, True, name="logits_long"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["matvec", "matvec", "rotary", "logits"])
    if op == "matvec":
        group = rng.choice([32, 64, 128])
        k = max(1, _log(rng, 256, 16384) // group) * group
        n = min(_log(rng, 65, 131072), (131072 * 4096) // k)
        return _matvec(_log(rng, 1, 16), n, k, group, rng.choice(["bf16", "f16"]), rng.random() < 0.5, rng.choice(["none", "none", "relu", "gelu", "silu"]),
                       rng.random() < 0.3, rng.random() < 0.3)
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 192, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4 * 2])
        heads = _log(rng, 1, 64)
        dtype = rng.choice(["bf16", "f16", "f32"])
        most = 8192 * 40 * 128 // (heads * dim * (2 if dtype == "f32" else 1))
        return _rotary(max(1, min(_log(rng, 1, 16384), most)), heads, rng.choice([0, 1, 8]), dim, rot, rng.choice(["half", "interleaved"]), dtype,
                       rng.choice(["none", "linear", "ntk", "ramp"]), _log(rng, 1024, 1 << 21), rng.random() < 0.4, rng.random() < 0.3)
    rows = _log(rng, 1, 128)
    vocab = min(_log(rng, 1001, 262144), 64 * 131072 // rows)
    return _logits(rows, vocab, _log(rng, 1, 65536), rng.choice(["bf16", "f16", "f32"]), rng.choice(["f32", "f32", "same"]), rng.choice([0, 7, 300]),
                   rng.random() < 0.6, rng.random() < 0.85)


# ---------------------------------------------------------------------------------------------------------- prepare
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _prepare_matvec(c, g):
    m, n, k, group, t = c["m"], c["n"], c["k"], c["group"], TYPES[c["dtype"]]
    s = {"X": torch.randn((m, k), device="cuda", generator=g).to(t)}
    # weights of a trained projection, quantised group by group: symmetric (signed, -8..7) or with a zero point (0..15)
    packed, scales, points = [], [], []
    for i in range(0, n, 16384):
        w = torch.randn((min(16384, n - i), k // group, group), device="cuda", generator=g).mul_(k ** -0.5)
        if c["zeros"]:
            w += 0.3 * k ** -0.5 * torch.randn((w.shape[0], k // group, 1), device="cuda", generator=g)
            lo, hi = w.amin(2, keepdim=True).clamp(max=0), w.amax(2, keepdim=True).clamp(min=0)
            sc = ((hi - lo) / 15).to(t)
            z = (-lo / sc.float()).round().clamp(0, 15)
            q = ((w / sc.float()).round_() + z).clamp_(0, 15)
            points.append(z.view(-1, k // group).to(torch.uint8))
        else:
            sc = (w.abs().amax(2, keepdim=True) / 7).to(t)
            q = (w / sc.float()).round_().clamp_(-8, 7)
        q = q.view(-1, k).to(torch.int16).bitwise_and_(15).to(torch.uint8)
        packed.append(q[:, 0::2] | (q[:, 1::2] << 4))          # two per byte, low nibble = even k
        scales.append(sc.view(-1, k // group))
    s["W"], s["scales"] = torch.cat(packed), torch.cat(scales)
    if c["zeros"]:
        z = torch.cat(points)
        if z.shape[1] % 2:
            z = torch.cat([z, torch.zeros_like(z[:, :1])], 1)  # rows of zero points are whole bytes
        s["zeros"] = z[:, 0::2] | (z[:, 1::2] << 4)            # two per byte, low nibble = even group
    if c["bias"]:
        s["bias"] = torch.randn(n, device="cuda", generator=g).to(t)
    if c["residual"]:
        s["C"] = torch.randn((m, n), device="cuda", generator=g).to(t)
    s["Y"] = torch.empty((m, n), dtype=t, device="cuda")
    return s


def _prepare_rotary(c, g):
    t = TYPES[c["dtype"]]
    # the heads to rotate are the first ones of each token's row; `extra` heads (the values) follow and stay out of it
    x = torch.randn((c["tokens"], c["heads"] + c["extra"], c["dim"]), device="cuda", generator=g).to(t)
    if c["tokens"] >= 1024:         # whole sequences
        first = torch.randint(0, max(1, c["far"] - c["tokens"]), (1,), device="cuda", generator=g)
        pos = first + torch.arange(c["tokens"], device="cuda")
    else:                           # one token of each sequence
        pos = torch.randint(0, c["far"], (c["tokens"],), device="cuda", generator=g)
    if c["padded"]:
        pos[c["tokens"] - c["tokens"] // 7:] = -1
    return {"x": x, "pos": pos, "y": torch.empty((c["tokens"], c["heads"], c["dim"]), dtype=t, device="cuda")}


def _prepare_logits(c, g):
    b, v, n = c["rows"], c["vocab"], c["history"]
    s = {"x": (torch.randn((b, v), device="cuda", generator=g) * 3).to(TYPES[c["dtype"]])}
    if c["penalties"]:
        # what was said so far: few frequent tokens and many rare ones, rows of different lengths behind which nothing is valid
        u = torch.rand((b, n), device="cuda", generator=g)
        s["history"] = ((v ** u).long() - 1 + torch.randint(0, v, (b, 1), device="cuda", generator=g)).remainder(v).int()
        length = (n - torch.randint(0, n + 1, (b,), device="cuda", generator=g) // 2).int()
        s["history"].masked_fill_(torch.arange(n, device="cuda") >= length[:, None], -1)
        s["length"] = length
        s["prompt"] = (length * torch.rand(b, device="cuda", generator=g)).int()
        s["repetition"] = 1 + torch.rand(b, device="cuda", generator=g)
        s["presence"] = torch.rand(b, device="cuda", generator=g)
        s["frequency"] = torch.rand(b, device="cuda", generator=g) * 0.5
    if c["biases"]:
        count = torch.randint(0, c["biases"] + 1, (b,), device="cuda", generator=g)
        s["bias_begin"] = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), count.cumsum(0)]).int()
        total = b * c["biases"]       # the list keeps room for the longest rows
        s["bias_ids"] = torch.randint(0, v, (total,), device="cuda", generator=g).int()
        s["bias_values"] = torch.randn(total, device="cuda", generator=g) * 5
    if c["mask"]:
        words = (v + 31) // 32
        share = torch.rand((b, 1), device="cuda", generator=g) ** 4      # most grammars allow little at a time
        allowed = torch.rand((b, words * 32), device="cuda", generator=g) < share
        if b > 2:
            allowed[2] = False                                            # a grammar that has come to its end
        weights = 1 << torch.arange(32, dtype=torch.int64, device="cuda")
        s["mask"] = (allowed.view(b, words, 32).long() * weights).sum(2).to(torch.int32)
    s["y"] = torch.empty((b, v), dtype=TYPES[c["dtype"] if c["out"] == "same" else c["out"]], device="cuda")
    return s


def prepare(case, seed):
    g = _generator(seed)
    s = {"matvec": _prepare_matvec, "rotary": _prepare_rotary, "logits": _prepare_logits}[case["op"]](case, g)
    s["case"] = case
    return s


# ------------------------------------------------------------------------------------------------------ plain forms
def _nibbles(p):
    return torch.stack([p & 15, p >> 4], 2).view(p.shape[0], -1)


def _activate(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "gelu":
        return v * 0.5 * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    return v


def _plain_matvec(s):
    c = s["case"]
    n, k, group = c["n"], c["k"], c["group"]
    q = _nibbles(s["W"])
    if c["zeros"]:
        q = q.float().view(n, -1, group) - _nibbles(s["zeros"])[:, :k // group, None].float()
    else:
        q = ((q ^ 8).float() - 8).view(n, -1, group)
    w = (q * s["scales"].float()[:, :, None]).view(n, k)
    y = s["X"].float() @ w.t()
    if c["residual"]:
        y = y + s["C"].float()
    if c["bias"]:
        y = y + s["bias"].float()
    return _activate(y, c["act"]).to(s["X"].dtype)


#: base, factor and the ramp's borders (rotations over the original length) that the scaled cases use
BASE, FACTOR, LOW, HIGH, ORIGINAL, RAMP_SCALE = 10000.0, 8.0, 1.0, 32.0, 8192, 0.1 * math.log(8.0) + 1


def _plain_frequencies(rot, scaling):
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    if scaling == "ntk":
        return (BASE * FACTOR ** (rot / (rot - 2))) ** (-2 * i / rot)
    f = BASE ** (-2 * i / rot)
    if scaling == "linear":
        return f / FACTOR
    if scaling == "ramp":
        keep = ((ORIGINAL * f / (2 * math.pi) - LOW) / (HIGH - LOW)).clamp(0, 1)
        return f * keep + f / FACTOR * (1 - keep)
    return f


def _plain_rotary(s):
    c = s["case"]
    rot, x = c["rot"], s["x"][:, :c["heads"]].float()
    angle = s["pos"].double()[:, None] * _plain_frequencies(rot, c["scaling"])         # far positions: 64 bits up to the sine
    scale = RAMP_SCALE if c["scaling"] == "ramp" else 1.0
    cos, sin = (torch.cos(angle) * scale).float()[:, None], (torch.sin(angle) * scale).float()[:, None]
    if c["backward"]:
        sin = -sin
    if c["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(2)
    y = torch.cat([turned, x[..., rot:]], -1)
    return torch.where((s["pos"] < 0)[:, None, None], x, y).to(s["x"].dtype)


def _plain_logits(s):
    c = s["case"]
    b, v = c["rows"], c["vocab"]
    x = s["x"].float()
    if c["penalties"]:
        at = torch.arange(c["history"], device="cuda")
        valid = at < s["length"][:, None]
        ids = torch.where(valid, s["history"], 0).long()
        seen = torch.zeros((b, v), device="cuda").scatter_add_(1, ids, valid.float())
        count = torch.zeros((b, v), device="cuda").scatter_add_(1, ids, (valid & (at >= s["prompt"][:, None])).float())
        r = s["repetition"][:, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - (s["frequency"][:, None] * count + s["presence"][:, None] * (count > 0))
    if c["biases"]:
        e = torch.arange(s["bias_ids"].shape[0], device="cuda")
        row = (e[:, None] >= s["bias_begin"][None, 1:]).sum(1)
        there = row < b
        flat = torch.where(there, row * v + s["bias_ids"].long(), 0)
        x = x + torch.zeros(b * v, device="cuda").scatter_add_(0, flat, torch.where(there, s["bias_values"], 0)).view(b, v)
    if c["mask"]:
        bit = (s["mask"][:, :, None] >> torch.arange(32, dtype=torch.int32, device="cuda")) & 1
        x = torch.where(bit.view(b, -1)[:, :v] == 0, -math.inf, x)
    return x.to(s["y"].dtype)


# ------------------------------------------------------------------------------------- the framework's own operators
_registry = None


def _plugin(c):
    """The w4a16 plugin for these rows: the registry's pick, or, where the output transform is asked for, the one that has it."""
    global _registry
    import sm120_gemm_b200 as lib

    if _registry is None:
        _registry = lib.KernelRegistry()
        _registry.load_dir(dt="w4a16")
    if c["act"] != "none" or c["bias"] or c["residual"]:
        return _registry.find("w4a16_bm128_bn%d_bk32_s8_cg1_sk1_ab1_e2" % (8 if c["m"] <= 8 else 16))
    return _registry.heuristic(c["m"], c["n"], c["k"], "w4a16")


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _matvec_call(s):
    import sm120_gemm_b200 as lib

    c, a = s["case"], lib.GemmArgs()
    a.M, a.N, a.K, a.group_size = c["m"], c["n"], c["k"], c["group"]
    a.x_dtype = TYPE_IDS[c["dtype"]]
    a.X, a.W, a.Y, a.w_scale, a.w_zero = _ptr(s["X"]), _ptr(s["W"]), _ptr(s["Y"]), _ptr(s["scales"]), _ptr(s.get("zeros"))
    a.bias, a.C, a.beta, a.activation = _ptr(s.get("bias")), _ptr(s.get("C")), float(c["residual"]), ACTS[c["act"]]
    kernel = _plugin(c)
    return lambda: lib.dispatch_ex(kernel, a), a, s["Y"]


def _rotary_call(s):
    import sm120_gemm_b200 as lib

    c, a = s["case"], lib.GemmRotaryArgs()
    a.dtype, a.layout, a.backward = TYPE_IDS[c["dtype"]], {"half": 0, "interleaved": 1}[c["layout"]], c["backward"]
    a.tokens, a.heads, a.head_dim, a.rot_dim = c["tokens"], c["heads"], c["dim"], c["rot"]
    a.x, a.y, a.positions = _ptr(s["x"]), _ptr(s["y"]), _ptr(s["pos"])
    a.x_token_stride, a.x_head_stride, a.y_token_stride, a.y_head_stride = s["x"].stride(0), s["x"].stride(1), s["y"].stride(0), s["y"].stride(1)
    a.base, a.scaling, a.factor = BASE, {"none": 0, "linear": 1, "ntk": 2, "ramp": 3}[c["scaling"]], FACTOR
    a.low_rotations, a.high_rotations, a.original_length = LOW, HIGH, ORIGINAL
    a.scale = RAMP_SCALE if c["scaling"] == "ramp" else 1.0
    return lambda: lib.rotary(a), a, s["y"]


def _logits_call(s):
    import sm120_gemm_b200 as lib

    c, a = s["case"], lib.GemmLogitsArgs()
    a.x_dtype, a.y_dtype = TYPE_IDS[c["dtype"]], TYPE_IDS[c["dtype"] if c["out"] == "same" else c["out"]]
    a.rows, a.vocab, a.x, a.y, a.x_ld, a.y_ld = c["rows"], c["vocab"], _ptr(s["x"]), _ptr(s["y"]), s["x"].stride(0), s["y"].stride(0)
    if c["penalties"]:
        a.history, a.history_ld, a.history_len, a.prompt_len = _ptr(s["history"]), s["history"].stride(0), _ptr(s["length"]), _ptr(s["prompt"])
        a.repetition, a.presence, a.frequency = _ptr(s["repetition"]), _ptr(s["presence"]), _ptr(s["frequency"])
    if c["biases"]:
        a.bias_ids, a.bias_values, a.bias_begin = _ptr(s["bias_ids"]), _ptr(s["bias_values"]), _ptr(s["bias_begin"])
    if c["mask"]:
        a.mask, a.mask_ld = _ptr(s["mask"]), s["mask"].stride(0)
    return lambda: lib.logits(a), a, s["y"]


def run(state):
    if not own:
        return {"matvec": _plain_matvec, "rotary": _plain_rotary, "logits": _plain_logits}[state["case"]["op"]](state)
    if "call" not in state:          # the argument block that a program fills once and uses for every token
        state["call"] = {"matvec": _matvec_call, "rotary": _rotary_call, "logits": _logits_call}[state["case"]["op"]](state)
    call, args, out = state["call"]
    args.stream = torch.cuda.current_stream().cuda_stream
    call()
    return out


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "matvec":
        m, n, k, groups = c["m"], c["n"], c["k"], c["k"] // c["group"]
        b = n * k / 2 + n * groups * 2 + m * k * 2 + m * n * 2
        b += n * ((groups + 1) // 2) if c["zeros"] else 0
        b += n * 2 if c["bias"] else 0
        b += m * n * 2 if c["residual"] else 0
        return {"bytes": b, "flops": 2.0 * m * n * k}
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if c["op"] == "rotary":
        values = c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 2.0 * values * size[c["dtype"]] + 8 * c["tokens"], "flops": 3.0 * c["tokens"] * c["heads"] * c["rot"]}
    values = c["rows"] * c["vocab"]
    b = values * (size[c["dtype"]] + size[c["dtype"] if c["out"] == "same" else c["out"]])
    b += c["rows"] * (0.75 * c["history"] * 4 + 20) if c["penalties"] else 0     # a row holds three quarters of the longest on average
    b += c["rows"] * (c["biases"] / 2 * 8 + 4) if c["biases"] else 0
    b += values / 8 if c["mask"] else 0
    return {"bytes": b, "flops": 4.0 * values}


# ------------------------------------------------------------------------------------------------------------ exact
def _exact_matvec(c, s):
    n, k, group = c["n"], c["k"], c["group"]
    x = s["X"].double()
    y = torch.empty((c["m"], n), dtype=torch.float64, device="cuda")
    for i in range(0, n, 8192):
        w = s["W"][i:i + 8192]
        full = torch.empty((w.shape[0], k), dtype=torch.float64, device="cuda")
        full[:, 0::2], full[:, 1::2] = w % 16, w // 16
        which = torch.arange(k, device="cuda") // group
        if c["zeros"]:
            z = s["zeros"][i:i + 8192]
            full -= ((z[:, which // 2] // (1 + 15 * (which % 2)).to(torch.uint8)) % 16).double()
        else:
            full = torch.where(full >= 8, full - 16, full)
        full *= s["scales"][i:i + 8192].double()[:, which]
        y[:, i:i + 8192] = torch.einsum("mk,nk->mn", x, full)
    if c["residual"]:
        y += s["C"].double()
    if c["bias"]:
        y += s["bias"].double()
    if c["act"] == "relu":
        y = y.clamp(min=0)
    elif c["act"] == "gelu":
        y = 0.5 * y * torch.special.erfc(-y / math.sqrt(2))
    elif c["act"] == "silu":
        y = y * torch.special.expit(y)
    return y


def _exact_rotary(c, s):
    rot, half = c["rot"], c["rot"] // 2
    x = s["x"][:, :c["heads"]].double()
    f = []
    for i in range(half):
        v = math.exp(-2 * i / rot * math.log(BASE))
        if c["scaling"] == "ntk":
            v = math.exp(-2 * i / rot * (math.log(BASE) + rot / (rot - 2) * math.log(FACTOR)))
        elif c["scaling"] == "linear":
            v /= FACTOR
        elif c["scaling"] == "ramp":
            turns = ORIGINAL * v / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - LOW) / (HIGH - LOW)))
            v = v * keep + v * (1 - keep) / FACTOR
        f.append(v)
    angle = s["pos"].double()[:, None] * torch.tensor(f, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(angle, RAMP_SCALE if c["scaling"] == "ramp" else 1.0), -angle if c["backward"] else angle)[:, None]
    turn = torch.where((s["pos"] < 0)[:, None, None], torch.ones_like(turn), turn)
    first = torch.arange(half, device="cuda") * (1 if c["layout"] == "half" else 2)
    second = first + (half if c["layout"] == "half" else 1)
    z = torch.complex(x[..., first], x[..., second]) * turn
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_logits(c, s):
    x = s["x"].double().cpu().numpy()
    for b in range(c["rows"]):
        row = x[b]
        if c["penalties"]:
            said = s["history"][b, :int(s["length"][b])].cpu().numpy()
            r, p, f = (float(s[k][b]) for k in ("repetition", "presence", "frequency"))
            every = np.unique(said)
            row[every] = np.where(row[every] > 0, row[every] / r, row[every] * r)
            ids, count = np.unique(said[int(s["prompt"][b]):], return_counts=True)
            row[ids] -= f * count + p
        if c["biases"]:
            lo, hi = int(s["bias_begin"][b]), int(s["bias_begin"][b + 1])
            np.add.at(row, s["bias_ids"][lo:hi].cpu().numpy(), s["bias_values"][lo:hi].double().cpu().numpy())
        if c["mask"]:
            bits = np.unpackbits(s["mask"][b].cpu().numpy().view(np.uint8), bitorder="little")[:c["vocab"]]
            row[bits == 0] = -np.inf
    return torch.from_numpy(x)


def exact(case, seed):
    s = prepare(case, seed)
    return {"matvec": _exact_matvec, "rotary": _exact_rotary, "logits": _exact_logits}[case["op"]](case, s)
