"""What is measured of the grouped linear and of the linear with an epilogue: cases, their plain form, their work.

Two families on MXFP8 operands (E4M3 values, one power-of-two scale per 32 values along the contraction):

  grouped   rows offsets[g] .. offsets[g + 1] - 1 of x belong to group g (an expert):  y[r] = q(x[r]) q(w[g])^T;
            backward: dx[r] = q(dy[r]) q(w[g]), dw[g] = q(dy_g)^T q(x_g), each operand quantized along its own
            contraction (the tokens of a group in blocks of 32 from the group's first row).
  epilogue  z = q(x) q(w)^T + bias, y = act(z) + residual; backward: dz = dy act'(z) with z and dz in BF16,
            dx = q(dz) q(w), dw = q(dz)^T q(x), dbias = sum of dz over the rows.
"""

import math

import torch

own = False

BLOCK = 32


# ------------------------------------------------------------------------------------------------ cases

def listed():
    g = {"head": 0, "tail": 0, "skew": 0.5, "pitch": 0}
    e = {"bias": True, "residual": False, "pitch": 0}
    return [
        # one decode step of a few sequences through small packed experts: the launches are the time
        {"name": "grouped_fwd_small", "op": "grouped_fwd", "t": 16, "groups": 8, "k": 1024, "n": 1024, "packed": True, **g},
        # decode of a batch: every expert's packed weight is streamed once for a handful of rows
        {"name": "grouped_fwd_decode", "op": "grouped_fwd", "t": 128, "groups": 32, "k": 4096, "n": 4096, "packed": True, **g},
        # prefill through packed experts, uneven routing
        {"name": "grouped_fwd_prefill", "op": "grouped_fwd", "t": 8192, "groups": 32, "k": 4096, "n": 2048, "packed": True,
         **{**g, "skew": 1.0}},
        # training forward: BF16 master weights, both operands quantized in the step
        {"name": "grouped_fwd_train", "op": "grouped_fwd", "t": 16384, "groups": 8, "k": 4096, "n": 4096, "packed": False, **g},
        # odd widths, rows of the batch before the first and behind the last group, x a slice of a wider tensor
        {"name": "grouped_fwd_odd", "op": "grouped_fwd", "t": 1003, "groups": 7, "k": 1000, "n": 1238, "packed": False,
         "head": 3, "tail": 21, "skew": 1.0, "pitch": 24},
        # training backward of the same experts
        {"name": "grouped_bwd_train", "op": "grouped_bwd", "t": 16384, "groups": 8, "k": 4096, "n": 4096, "packed": False, **g},
        # backward of a small uneven batch, odd widths
        {"name": "grouped_bwd_odd", "op": "grouped_bwd", "t": 777, "groups": 12, "k": 520, "n": 776, "packed": False,
         "head": 0, "tail": 9, "skew": 1.0, "pitch": 0},
        # decode through a packed projection with bias and residual
        {"name": "epilogue_fwd_small", "op": "epilogue_fwd", "m": 8, "k": 1024, "n": 1024, "act": "silu", "packed": True,
         **{**e, "residual": True}},
        # up projection of a feed-forward block in a training batch, BF16 weight
        {"name": "epilogue_fwd_up", "op": "epilogue_fwd", "m": 8192, "k": 4096, "n": 14336, "act": "gelu", "packed": False, **e},
        # its down projection in a serving batch: packed weight, residual added
        {"name": "epilogue_fwd_down", "op": "epilogue_fwd", "m": 8192, "k": 14336, "n": 4096, "act": "none", "packed": True,
         **{**e, "residual": True}},
        # training step of one projection
        {"name": "epilogue_train", "op": "epilogue_train", "m": 8192, "k": 4096, "n": 8192, "act": "gelu", "packed": False,
         **{**e, "residual": True}},
        # training step of a ragged batch, odd widths
        {"name": "epilogue_train_odd", "op": "epilogue_train", "m": 517, "k": 712, "n": 1001, "act": "relu2", "packed": False,
         **{**e, "pitch": 8}},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["grouped_fwd", "grouped_fwd", "grouped_bwd", "epilogue_fwd", "epilogue_fwd", "epilogue_train"])
    k, n = _log(rng, 64, 8192), _log(rng, 64, 8192)
    if rng.random() < 0.6:
        k, n = max(128, k // 128 * 128), max(128, n // 128 * 128)
    pitch = rng.choice([0, 0, 8, 13])
    if op.startswith("grouped"):
        c = {"op": op, "t": _log(rng, 1, 16384), "groups": _log(rng, 1, 64), "k": k, "n": n,
             "packed": op == "grouped_fwd" and n % 128 == 0 and rng.random() < 0.6,
             "head": rng.choice([0, 0, 5]), "tail": rng.choice([0, 0, 17]), "skew": rng.choice([0.0, 0.5, 1.5]), "pitch": pitch}
        while c["groups"] * k * n > 8 * 4096 * 4096 or c["t"] * k * n > 16384 * 4096 * 4096:
            c["groups"], c["t"] = max(1, c["groups"] // 2), max(1, c["t"] // 2)
        return c
    c = {"op": op, "m": _log(rng, 1, 8192), "k": k, "n": n,
         "act": rng.choice(["none", "relu", "relu2", "silu", "gelu", "gelu_tanh"]),
         "packed": op == "epilogue_fwd" and rng.random() < 0.5, "bias": rng.random() < 0.8, "residual": rng.random() < 0.5,
         "pitch": pitch}
    while c["m"] * k * n > 8192 * 4096 * 8192:
        c["m"] //= 2
    return c


# ------------------------------------------------------------------------------------------------ inputs

def _wide(gen, rows, cols, pitch):
    """A [rows, cols] BF16 activation: normal values, one in a thousand fifty times larger; with `pitch` a slice of a
    wider tensor."""
    x = torch.randn(rows, cols + pitch, generator=gen, device="cuda")
    x = torch.where(torch.rand(rows, cols + pitch, generator=gen, device="cuda") < 0.001, 50.0 * x, x)
    return x.bfloat16()[:, :cols]


def _weight(gen, *shape):
    """A BF16 weight of the usual initial size."""
    return (torch.randn(*shape, generator=gen, device="cuda") / math.sqrt(shape[-1])).bfloat16()


def _packed(w):
    """A BF16 weight [..., N, K] as a checkpoint holds it: E4M3 bytes and the scale bytes in 128-row tiles
    (byte (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4 of tile [row / 128][block / 4])."""
    k = w.shape[-1]
    rows = w.numel() // k
    values, exponents = _blocks(w.reshape(rows, k).float())
    nb = exponents.shape[1]
    quotient = values * _pow2(-exponents).unsqueeze(-1)
    chunks = (nb + 3) // 4
    tiles = torch.zeros((rows + 127) // 128 * chunks * 512, dtype=torch.uint8, device=w.device)
    r = torch.arange(rows, device=w.device).unsqueeze(1)
    b = torch.arange(nb, device=w.device).unsqueeze(0)
    at = ((r // 128) * chunks + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4
    tiles[at.reshape(-1)] = (exponents + 127).to(torch.uint8).reshape(-1)
    return quotient.reshape(rows, nb * BLOCK).to(torch.float8_e4m3fn), tiles


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    k, n = case["k"], case["n"]
    if case["op"].startswith("grouped"):
        host = torch.Generator().manual_seed(seed)
        share = torch.softmax(case["skew"] * torch.randn(case["groups"], generator=host), 0)
        counts = torch.bincount(torch.multinomial(share, case["t"], replacement=True, generator=host), minlength=case["groups"])
        ends = torch.cumsum(counts, 0) + case["head"]
        offsets = torch.cat([torch.tensor([case["head"]]), ends])
        rows = case["head"] + case["t"] + case["tail"]
        s.update(counts=counts.tolist(), most=int(counts.max()), offsets=offsets.to(torch.int32).cuda(),
                 x=_wide(gen, rows, k, case["pitch"]), w=_weight(gen, case["groups"], n, k))
        if case["op"] == "grouped_bwd":
            s["dy"] = (0.1 * torch.randn(rows, n, generator=gen, device="cuda")).bfloat16()
    else:
        m = case["m"]
        s.update(x=_wide(gen, m, k, case["pitch"]), w=_weight(gen, n, k))
        s["b"] = torch.randn(n, generator=gen, device="cuda").bfloat16() if case["bias"] else None
        s["r"] = torch.randn(m, n, generator=gen, device="cuda").bfloat16() if case["residual"] else None
        if case["op"] == "epilogue_train":
            s["dy"] = (0.1 * torch.randn(m, n, generator=gen, device="cuda")).bfloat16()
            for name in ("x", "w", "b"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    if case["packed"]:
        q, scales = _packed(s["w"])
        if own:  # the handle that a serving program keeps of its packed weight: the same bytes, no work
            from rtx_b200.formats import make_mxfp8_tensor

            s["w"] = make_mxfp8_tensor(q, scales, tuple(s["w"].shape), "mma128")
        else:
            s.update(w=None, q=q, scales=scales)
    return s


# ------------------------------------------------------------------------------------------------ plain form

def _pow2(e):
    """2^e in FP32 from its exponent bits (e in -126 .. 127)."""
    return ((e + 127) << 23).view(torch.float32)


def _blocks(v):
    """v [..., K] in FP32 -> (the values MXFP8 holds, [..., blocks, 32]; the blocks' scale exponents)."""
    v = torch.nn.functional.pad(v, (0, -v.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    bits = v.abs().amax(-1).view(torch.int32)
    e = (bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000).int()  # the scale that brings the largest below 448
    e = e.clamp(min=-126)
    scale = _pow2(e).unsqueeze(-1)
    u = v * _pow2(-e).unsqueeze(-1)
    step = _pow2(((u.abs().view(torch.int32) >> 23) - 127).clamp(min=-6) - 3)  # three mantissa bits, 2^-9 at the least
    return torch.round(u / step) * step * scale, e


def _mx(v):
    """The FP32 values of v after MXFP8 quantization along the last dimension (which is padded to blocks)."""
    return _blocks(v.float())[0].flatten(-2)


def _unpack(q, scales, shape):
    """FP32 values of a packed weight, [..., padded K]."""
    rows, kp = q.shape
    nb = kp // BLOCK
    chunks = (nb + 3) // 4
    r = torch.arange(rows, device=q.device).unsqueeze(1)
    b = torch.arange(nb, device=q.device).unsqueeze(0)
    e = scales[((r // 128) * chunks + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4].int() - 127
    return (q.float().unflatten(-1, (nb, BLOCK)) * _pow2(e).unsqueeze(-1)).reshape(*shape[:-1], kp)


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0.0)
    if act == "relu2":
        return z.clamp(min=0.0).square()
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0.0).to(z.dtype)
    if act == "relu2":
        return 2.0 * z.clamp(min=0.0)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * z * z)
    return torch.ones_like(z)


def _places(s, rows):
    """For the groups padded to one length (whole blocks): the row of x behind each place, and the place behind each row
    of x; rows and places without a partner point at one past the end."""
    length = max(BLOCK, -(-s["most"] // BLOCK) * BLOCK)
    first, last = s["offsets"][:-1].long().unsqueeze(1), s["offsets"][1:].long().unsqueeze(1)
    row = first + torch.arange(length, device=first.device).unsqueeze(0)
    live = row < last
    row = torch.where(live, row, rows)
    place = torch.full((rows + 1,), row.numel(), device=row.device)
    place[row.reshape(-1)] = torch.arange(row.numel(), device=row.device)
    place[rows] = row.numel()
    return row, place[:rows]


def _spread(v, row):
    """[rows, c] -> [groups, length, c], zero behind each group's last row."""
    return torch.cat([v, v.new_zeros(1, v.shape[1])])[row]


def _gather(v, place):
    """[groups, length, c] -> [rows, c], zero in rows of no group."""
    v = v.flatten(0, 1)
    return torch.cat([v, v.new_zeros(1, v.shape[1])])[place]


def _plain_grouped(s):
    x, k, n = s["x"], s["k"], s["n"]
    row, place = _places(s, x.shape[0])
    if s["op"] == "grouped_fwd":
        w = _unpack(s["q"], s["scales"], (s["groups"], n, k)) if s["packed"] else _mx(s["w"])
        return _gather(torch.bmm(_spread(_mx(x), row), w.transpose(1, 2)), place).bfloat16()
    dy, w = s["dy"], s["w"]
    w_t = _mx(w.transpose(1, 2))
    dx = _gather(torch.bmm(_spread(_mx(dy), row), w_t.transpose(1, 2)), place)
    dy_t = _mx(_spread(dy, row).transpose(1, 2))
    x_t = _mx(_spread(x, row).transpose(1, 2))
    return {"dx": dx.bfloat16(), "dw": torch.bmm(dy_t, x_t.transpose(1, 2)).bfloat16()}


def _plain_epilogue(s):
    x, act = s["x"].detach(), s["act"]
    w = _unpack(s["q"], s["scales"], (s["n"], s["k"])) if s["packed"] else _mx(s["w"].detach())
    z = _mx(x) @ w.t()
    if s["b"] is not None:
        z = z + s["b"].detach().float()
    y = _act(z, act)
    y = (y if s["r"] is None else y + s["r"].float()).bfloat16()
    if s["op"] == "epilogue_fwd":
        return y
    dz = s["dy"].float()
    if act != "none":
        dz = (dz.double() * _slope(z.bfloat16().double(), act)).float()  # in 64 bits: the product is rounded to 8 bits next
    dzq = dz.bfloat16()
    dx = _mx(dzq) @ _mx(s["w"].detach().t()).t()
    dw = _mx(dzq.t()) @ _mx(x.t()).t()
    return {"y": y, "dx": dx.bfloat16(), "dw": dw.bfloat16(), "db": None if s["b"] is None else dz.sum(0).bfloat16()}


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    if own:
        import rtx_b200

        if s["op"] == "grouped_fwd":
            return rtx_b200.mxfp8_grouped_linear(s["x"], s["w"], s["offsets"])
        if s["op"] == "grouped_bwd":
            dx, dw = rtx_b200.mxfp8_grouped_linear_backward(s["dy"], s["x"], s["w"], s["offsets"])
            return {"dx": dx, "dw": dw}
        y = rtx_b200.mxfp8_linear_epilogue(s["x"], s["w"], s["b"], s["r"], activation=s["act"])
        if s["op"] == "epilogue_fwd":
            return y
        leaves = [s["x"], s["w"]] + ([] if s["b"] is None else [s["b"]])
        grads = torch.autograd.grad(y, leaves, s["dy"])
        return {"y": y, "dx": grads[0], "dw": grads[1], "db": None if s["b"] is None else grads[2]}
    return _plain_grouped(s) if s["op"].startswith("grouped") else _plain_epilogue(s)


def work(case):
    k, n = case["k"], case["n"]
    if case["op"].startswith("grouped"):
        t, groups = case["t"], min(case["groups"], case["t"])
        held = 33 / 32 if case["packed"] else 2
        if case["op"] == "grouped_fwd":
            return {"bytes": 2 * t * k + held * groups * n * k + 2 * (t + case["head"] + case["tail"]) * n, "flops": 2 * t * n * k}
        rows = t + case["head"] + case["tail"]
        return {"bytes": 2 * t * (k + n) + 2 * groups * n * k + 2 * rows * k + 2 * case["groups"] * n * k, "flops": 4 * t * n * k}
    m = case["m"]
    held = 33 / 32 if case["packed"] else 2
    size = 2 * m * k + held * n * k + 2 * m * n + (2 * n if case["bias"] else 0) + (2 * m * n if case["residual"] else 0)
    if case["op"] == "epilogue_fwd":
        return {"bytes": size, "flops": 2 * m * n * k}
    return {"bytes": size + 2 * m * n + 2 * m * k + 2 * n * k + (2 * n if case["bias"] else 0), "flops": 6 * m * n * k}


# ------------------------------------------------------------------------------------------------ 64 bits

def _two64(p):
    """2^p in 64 bits from its exponent bits."""
    return ((p.long() + 1023) << 52).view(torch.float64)


def _mx64(v):
    """MXFP8 values of v along its last dimension, in 64 bits: with the largest of a block written f 2^p, 1/2 <= f < 1, the
    scale is 2^(p - 9), doubled where f > 7/8; a value u 2^q of the scaled block keeps four significant bits, and none
    below 2^-9."""
    v = v.double()
    short = -v.shape[-1] % 32
    if short:
        v = torch.cat([v, v.new_zeros(*v.shape[:-1], short)], -1)
    b = v.reshape(*v.shape[:-1], -1, 32)
    f, p = torch.frexp(b.abs().max(-1, keepdim=True).values)
    scale = _two64(((p - 9) + (f > 0.875).to(p.dtype)).clamp(min=-126))
    u = b / scale
    q = torch.frexp(u)[1]
    unit = _two64((q - 4).clamp(min=-9))
    return (torch.round(u / unit) * unit * scale).reshape(v.shape)


def exact(case, seed):
    s = prepare({**case, "packed": False}, seed)
    w = s["w"].detach()
    x = s["x"].detach()
    if case["op"].startswith("grouped"):
        at = s["offsets"].tolist()
        spans = [(g, at[g], at[g + 1]) for g in range(case["groups"]) if at[g + 1] > at[g]]
        if case["op"] == "grouped_fwd":
            y = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device=x.device)
            for g, a, b in spans:
                y[a:b] = _mx64(x[a:b]) @ _mx64(w[g]).T
            return y
        dy = s["dy"]
        dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
        dw = torch.zeros(w.shape, dtype=torch.float64, device=x.device)
        for g, a, b in spans:
            dx[a:b] = _mx64(dy[a:b]) @ _mx64(w[g].T).T
            dw[g] = _mx64(dy[a:b].T) @ _mx64(x[a:b].T).T
        return {"dx": dx, "dw": dw}
    z = _mx64(x) @ _mx64(w).T
    if s["b"] is not None:
        z += s["b"].detach().double()
    shape = {
        "none": lambda v: v,
        "relu": torch.relu,
        "relu2": lambda v: torch.relu(v) ** 2,
        "silu": lambda v: v * torch.sigmoid(v),
        "gelu": lambda v: 0.5 * v * torch.erfc(-v / math.sqrt(2.0)),
        "gelu_tanh": lambda v: v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)),
    }[case["act"]]
    y = shape(z)
    if s["r"] is not None:
        y = y + s["r"].double()
    if case["op"] == "epilogue_fwd":
        return y
    dz = s["dy"].double()
    if case["act"] != "none":
        with torch.enable_grad():
            v = z.bfloat16().double().requires_grad_(True)
            dz = dz * torch.autograd.grad(shape(v).sum(), v)[0]
    held = dz.bfloat16()
    return {"y": y, "dx": _mx64(held) @ _mx64(w.T).T, "dw": _mx64(held.T) @ _mx64(x.T).T,
            "db": None if s["b"] is None else dz.sum(0)}
