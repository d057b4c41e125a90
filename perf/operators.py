"""The RMS norm, the gated feed-forward block and the 8-bit product, as cases that can be timed and compared.

A case is a dict of plain values with a "kind":

  norm        residual addition and RMS norm, as a forward pass without gradients makes it: the sum, and the normalised rows in
              bfloat16 or (out8) in e4m3 with a scale for each row and 128 columns
  norm-train  the same with the bfloat16 output, and its backward pass
  gated       gate and up projection, activation and product, as a forward pass without gradients makes it
  gated-train the same with both pre-activations kept, and the backward pass from the gradient of the block's output
  product8    a linear layer in e4m3: the rows quantised (unless they are there already), the product with a weight that has a
              scale for each 128 x 128 tile, and the residual

Rows are tokens, D is the model's width, F the block's hidden width.  prepare() makes a case's inputs from the seed and what a
program keeps (weights, buffers, the down projection's transposed copy, which both sides read); run() is one pass.  The packed weight's
transposed copy, which only the framework's backward pass reads, is made in the pass: the weights change with every step.
"""
import math

import torch

own = False

BF16, F32, F64, F8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
GROUP = 128            # columns (and, of weights, rows) that share a scale
LARGEST = 448.0        # of e4m3
LEAST_SCALE = 2.0 ** -100
EPS = 1e-6
ACTIVATIONS = {"silu": 0, "gelu": 1}


def listed():
    return [
        # One new token's row on its way into an 8-bit projection.
        dict(name="norm-token", kind="norm", rows=1, D=1024, out8=True),
        # A long prompt's or an evaluation batch's rows into 8-bit projections, at the widest model.
        dict(name="norm-out8", kind="norm", rows=16384, D=2048, out8=True),
        # The headline model's batch (16 sequences of 1024 tokens, width 768) in a training step.
        dict(name="norm-train-d768", kind="norm-train", rows=16384, D=768),
        # Rows and columns that nothing divides: the tail of a corpus at an odd width.
        dict(name="norm-train-odd", kind="norm-train", rows=997, D=1000),
        # One token through the block: both matrices are read for it.
        dict(name="gated-token", kind="gated", tokens=1, D=1024, F=2816, act="silu"),
        # A ragged batch of short texts scored at once.
        dict(name="gated-odd", kind="gated", tokens=333, D=640, F=1720, act="silu"),
        # The headline model's batch with a gated block of the same parameter count as its MLP.
        dict(name="gated-train-d768", kind="gated-train", tokens=16384, D=768, F=2048, act="silu"),
        # The long-context model's batch (4 sequences of 4096 tokens, width 1024, hidden width 4096), GELU gate.
        dict(name="gated-train-d1024", kind="gated-train", tokens=16384, D=1024, F=4096, act="gelu"),
        # One token through a layer that widens.
        dict(name="product8-token", kind="product8", tokens=1, K=1024, N=4096, rows8=False, residual=False),
        # A batch of sequences one token each, through a layer that narrows.
        dict(name="product8-batch", kind="product8", tokens=64, K=4096, N=1024, rows8=True, residual=True),
        # Sizes that neither tiles nor scale blocks divide.
        dict(name="product8-odd", kind="product8", tokens=777, K=1904, N=1000, rows8=False, residual=True),
        # A long prompt or an evaluation batch.
        dict(name="product8-large", kind="product8", tokens=16384, K=4096, N=4096, rows8=False, residual=True),
    ]


def _spread(rng, low, high, step=1):
    """A multiple of `step` from low to high, spread over the logarithm."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high, max(low, int(round(value / step)) * step))


def draw(rng):
    """One more case of the ranges above."""
    kind = rng.choice(["norm", "norm-train", "gated", "gated-train", "product8", "product8"])
    if kind == "norm":
        return dict(kind=kind, rows=_spread(rng, 1, 16384), D=_spread(rng, 64, 2048, 8), out8=rng.choice([True, True, False]))
    if kind == "norm-train":
        return dict(kind=kind, rows=_spread(rng, 1, 16384), D=_spread(rng, 64, 2048, 8))
    if kind == "gated":
        return dict(kind=kind, tokens=_spread(rng, 1, 16384), D=_spread(rng, 64, 1024, 8), F=_spread(rng, 128, 4096, 8),
                    act=rng.choice(["silu", "gelu"]))
    if kind == "gated-train":
        return dict(kind=kind, tokens=_spread(rng, 128, 16384), D=_spread(rng, 128, 1024, 8), F=_spread(rng, 256, 4096, 8),
                    act=rng.choice(["silu", "gelu"]))
    return dict(kind=kind, tokens=_spread(rng, 1, 16384), K=_spread(rng, 128, 4096, 16), N=_spread(rng, 128, 4096, 8),
                rows8=rng.choice([True, False]), residual=rng.choice([True, False]))


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _normal(generator, *shape, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=generator) * scale).to(BF16)


def _rows(generator, rows, columns):
    """Activations: normal, with a few columns much larger than the others, as a residual stream has them."""
    weight = torch.ones(columns, device="cuda")
    weight[torch.rand(columns, device="cuda", generator=generator) < 0.01] = 12.0
    return (torch.randn(rows, columns, device="cuda", generator=generator) * weight).to(BF16)


def _empty(*shape, dtype=BF16):
    return torch.empty(*shape, device="cuda", dtype=dtype)


def _groups(n):
    return -(-n // GROUP)


def _tile_codes(w):
    """A weight as a program holds it in 8 bits: its codes, and a scale for each 128 x 128 tile."""
    n, k = w.shape
    padded = torch.zeros(_groups(n) * GROUP, _groups(k) * GROUP, device="cuda")
    padded[:n, :k] = w
    tiles = padded.view(_groups(n), GROUP, _groups(k), GROUP)
    scale = (tiles.abs().amax((1, 3)) / LARGEST).clamp(min=LEAST_SCALE)
    codes = (tiles / scale[:, None, :, None]).to(F8).view(padded.shape)
    return codes[:n, :k].contiguous(), scale


def _row_codes(x):
    m, k = x.shape
    padded = torch.zeros(m, _groups(k) * GROUP, device="cuda")
    padded[:, :k] = x
    groups = padded.view(m, _groups(k), GROUP)
    scale = (groups.abs().amax(2) / LARGEST).clamp(min=LEAST_SCALE)
    codes = (groups / scale[:, :, None]).to(F8).view(m, -1)
    return codes[:, :k].contiguous(), scale.t().contiguous()


def _gamma(generator, columns):
    """The norm's weight, and the two 16-bit halves that the framework holds of it."""
    gamma = 1 + 0.1 * torch.randn(columns, device="cuda", generator=generator)
    bits = gamma.view(torch.int32)
    return gamma, (bits >> 16).to(torch.int16), (bits & 0xffff).to(torch.int32).to(torch.int16)


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    kind = case["kind"]
    if kind in ("norm", "norm-train"):
        m, d = case["rows"], case["D"]
        gamma, high, low = _gamma(generator, d)
        s = dict(kind=kind, m=m, d=d, x=_rows(generator, m, d), residual=_rows(generator, m, d), gamma=gamma, high=high, low=low,
                 sum=_empty(m, d))
        if kind == "norm-train":
            s |= dict(y=_empty(m, d), dy=_normal(generator, m, d), dsum=_normal(generator, m, d), dx=_empty(m, d),
                      dgamma=_empty(d, dtype=F32))
        elif case["out8"]:
            s |= dict(q=_empty(m, d, dtype=F8), scales=_empty(_groups(d), m, dtype=F32))
        else:
            s |= dict(y=_empty(m, d))
        return s
    if kind in ("gated", "gated-train"):
        m, d, f = case["tokens"], case["D"], case["F"]
        s = dict(kind=kind, m=m, d=d, f=f, act=case["act"], x=_normal(generator, m, d),
                 w=_normal(generator, 2 * f, d, scale=d ** -0.5), h=_empty(m, f))
        if kind == "gated-train":
            down = _normal(generator, d, f, scale=f ** -0.5)
            s |= dict(w_t=s["w"].t().contiguous(), down_t=down.t().contiguous(), dy=_normal(generator, m, d),
                      gu=_empty(m, 2 * f), dgu=_empty(m, 2 * f), dx=_empty(m, d))
        return s
    m, k, n = case["tokens"], case["K"], case["N"]
    x = _rows(generator, m, k)
    w, w_scales = _tile_codes(_normal(generator, n, k, scale=k ** -0.5))
    s = dict(kind=kind, m=m, k=k, n=n, x=x, w=w, w_scales=w_scales, rows8=case["rows8"], y=_empty(m, n),
             residual=_normal(generator, m, n) if case["residual"] else None)
    if case["rows8"]:
        s["q"], s["scales"] = _row_codes(x)
    else:
        s |= dict(q=_empty(m, k, dtype=F8), scales=_empty(_groups(k), m, dtype=F32))
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------


def _act(g, act):
    if act == "silu":
        return g / (1 + torch.exp(-g))
    return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))


def _act_slope(g, act):
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return s * (1 + g * (1 - s))
    return 0.5 * (1 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def _quantized(v):
    """Rows of 32-bit values: e4m3 codes, and scales [group][row]."""
    m, k = v.shape
    wide = torch.nn.functional.pad(v, (0, -k % GROUP)).view(m, -1, GROUP)
    scale = (wide.abs().amax(2) / LARGEST).clamp(min=LEAST_SCALE)
    return (wide / scale[:, :, None]).view(m, -1)[:, :k].to(F8), scale.t().contiguous()


def _plain(s):
    kind = s["kind"]
    if kind in ("norm", "norm-train"):
        h = (s["x"].float() + s["residual"].float()).to(BF16)
        wide = h.float()
        r = torch.rsqrt(wide.square().mean(1, keepdim=True) + EPS)
        v = wide * r * s["gamma"]
        if kind == "norm" and "q" in s:
            q, scales = _quantized(v)
            return dict(sum=h, q=q, scales=scales)
        if kind == "norm":
            return dict(sum=h, y=v.to(BF16))
        t = s["dy"].float()
        g = t * s["gamma"]
        dx = r * g - wide * (r ** 3 * (wide * g).mean(1, keepdim=True))
        return dict(sum=h, y=v.to(BF16), dx=(s["dsum"].float() + dx).to(BF16), dgamma=(t * wide * r).sum(0))
    if kind in ("gated", "gated-train"):
        both = s["x"].float() @ s["w"].float().t()
        g, u = both[:, :s["f"]], both[:, s["f"]:]
        h = (_act(g, s["act"]) * u).to(BF16)
        if kind == "gated":
            return dict(h=h)
        kept = both.to(BF16)
        g, u = kept[:, :s["f"]].float(), kept[:, s["f"]:].float()
        dh = s["dy"].float() @ s["down_t"].float().t()
        dgu = torch.cat([dh * u * _act_slope(g, s["act"]), dh * _act(g, s["act"])], 1)
        return dict(h=h, gu=kept, dgu=dgu.to(BF16), dx=(dgu @ s["w"].float()).to(BF16))
    if s["rows8"]:
        q, scales = s["q"], s["scales"]
    else:
        q, scales = _quantized(s["x"].float())
    x = q.float() * scales.t().repeat_interleave(GROUP, 1)[:, :s["k"]]
    w_scales = s["w_scales"].repeat_interleave(GROUP, 0).repeat_interleave(GROUP, 1)
    y = x @ (s["w"].float() * w_scales[:s["n"], :s["k"]]).t()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return dict(y=y.to(BF16)) if s["rows8"] else dict(y=y.to(BF16), q=q, scales=scales)


def _transpose(s, lib, stream):
    """The packed weight's transposed copy, by the framework's entry where it takes the shape."""
    w, w_t = s["w"], s["w_t"]
    rows, columns = w.shape
    if rows % 64 or columns % 64:
        w_t.copy_(w.t())
        return
    tiles = rows // 64 * (columns // 64)
    if "transpose" not in s:  # one matrix: {int64 offset; int32 rows, columns, first tile, 0}
        s["transpose"] = torch.tensor([0, rows | columns << 32, 0], device="cuda")
    from turbogpt_amd.bridge import check
    check(lib.tgk_transpose_batch(stream, w.data_ptr(), w_t.data_ptr(), s["transpose"].data_ptr(), 1, tiles))


def _own(s):
    from turbogpt_amd.bridge import check, library
    lib, kind, m = library(), s["kind"], s["m"]
    stream = torch.cuda.current_stream().cuda_stream
    if kind in ("norm", "norm-train"):
        d = s["d"]
        y = s["y"].data_ptr() if "y" in s else None
        q, scales = (s["q"].data_ptr(), s["scales"].data_ptr()) if "q" in s else (None, None)
        check(lib.tgk_rmsnorm_fwd(stream, m, d, s["x"].data_ptr(), s["residual"].data_ptr(), s["high"].data_ptr(),
                                  s["low"].data_ptr(), s["sum"].data_ptr(), y, q, scales, m, EPS))
        if kind == "norm":
            return dict(sum=s["sum"], q=s["q"], scales=s["scales"]) if q else dict(sum=s["sum"], y=s["y"])
        if "workspace" not in s:
            s["workspace"] = _empty(lib.tgk_rmsnorm_bwd_workspace(m, d), dtype=torch.uint8)
        check(lib.tgk_rmsnorm_bwd(stream, m, d, s["sum"].data_ptr(), s["dy"].data_ptr(), s["high"].data_ptr(),
                                  s["low"].data_ptr(), s["dsum"].data_ptr(), s["dx"].data_ptr(), s["dgamma"].data_ptr(), EPS, 0,
                                  s["workspace"].data_ptr(), s["workspace"].numel()))
        return dict(sum=s["sum"], y=s["y"], dx=s["dx"], dgamma=s["dgamma"])
    if kind in ("gated", "gated-train"):
        d, f, act = s["d"], s["f"], ACTIVATIONS[s["act"]]
        train = kind == "gated-train"
        check(lib.tgk_gated_fwd(stream, m, f, d, s["x"].data_ptr(), d, s["w"].data_ptr(), d, s["h"].data_ptr(), f,
                                s["gu"].data_ptr() if train else None, 2 * f, act))
        if not train:
            return dict(h=s["h"])
        _transpose(s, lib, stream)  # the weights are new in every step
        check(lib.tgk_gated_bwd(stream, m, f, d, s["dy"].data_ptr(), d, s["down_t"].data_ptr(), d, s["gu"].data_ptr(), 2 * f,
                                s["dgu"].data_ptr(), 2 * f, s["w_t"].data_ptr(), 2 * f, s["dx"].data_ptr(), d, act))
        return dict(h=s["h"], gu=s["gu"], dgu=s["dgu"], dx=s["dx"])
    k, n, residual = s["k"], s["n"], s["residual"]
    if not s["rows8"]:
        check(lib.tgk_quantize_rows(stream, m, k, s["x"].data_ptr(), k, s["q"].data_ptr(), k, s["scales"].data_ptr(), m))
    check(lib.tgk_gemm_q8(stream, m, n, k, s["q"].data_ptr(), k, s["scales"].data_ptr(), m, s["w"].data_ptr(), k,
                          s["w_scales"].data_ptr(), s["w_scales"].shape[1], s["y"].data_ptr(), n,
                          residual.data_ptr() if residual is not None else None, n))
    return dict(y=s["y"]) if s["rows8"] else dict(y=s["y"], q=s["q"], scales=s["scales"])


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm-train"):
        m, d = case["rows"], case["D"]
        if kind == "norm":
            out = m * d + 4 * m * _groups(d) if case["out8"] else 2 * m * d
            return dict(bytes=6 * m * d + 4 * d + out, flops=6.0 * m * d)
        return dict(bytes=(8 + 6) * m * d + 8 * d, flops=20.0 * m * d)  # x, residual, sum, y; dy, the sum's gradient, dx
    if kind in ("gated", "gated-train"):
        m, d, f = case["tokens"], case["D"], case["F"]
        if kind == "gated":
            return dict(bytes=2 * (m * d + 2 * f * d + m * f), flops=4.0 * m * f * d)
        # x, dy, dx; h, both pre-activations, their gradients; the three matrices
        return dict(bytes=2 * (3 * m * d + 5 * m * f + 3 * f * d), flops=10.0 * m * f * d)
    m, k, n = case["tokens"], case["K"], case["N"]
    rows = (1 if case["rows8"] else 3) * m * k + 4 * m * _groups(k)
    return dict(bytes=rows + n * k + 4 * _groups(n) * _groups(k) + (4 if case["residual"] else 2) * m * n, flops=2.0 * m * n * k)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------


def _nearest_e4m3(v):
    """The e4m3 values nearest to 64-bit ones of at most 448, ties to the even code: three mantissa bits from 2^-6 up, steps of
    2^-9 below."""
    _, exponent = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (exponent - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _scaled_groups(v):
    """(values of the codes, scales [group][row]) of 64-bit rows."""
    codes, scales = torch.empty_like(v), []
    for first in range(0, v.shape[1], GROUP):
        part = v[:, first:first + GROUP]
        scale = torch.clamp(part.abs().max(1).values / LARGEST, min=LEAST_SCALE)
        codes[:, first:first + GROUP] = _nearest_e4m3(part / scale[:, None])
        scales.append(scale)
    return codes, torch.stack(scales)


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind in ("norm", "norm-train"):
        total = (s["x"].to(F64) + s["residual"].to(F64)).to(BF16).to(F64)  # the sum is held, and read again, in bfloat16
        gamma = s["gamma"].to(F64)
        deviation = torch.sqrt((total * total).sum(1) / s["d"] + EPS)[:, None]
        unit = total / deviation
        if kind == "norm" and case["out8"]:
            codes, scales = _scaled_groups(unit * gamma)
            return dict(sum=total, q=codes, scales=scales)
        if kind == "norm":
            return dict(sum=total, y=unit * gamma)
        dy = s["dy"].to(F64)
        t = dy * gamma
        dx = (t - unit * (unit * t).sum(1, keepdim=True) / s["d"]) / deviation
        return dict(sum=total, y=unit * gamma, dx=s["dsum"].to(F64) + dx, dgamma=(dy * unit).sum(0))
    if kind in ("gated", "gated-train"):
        f = s["f"]
        x, w = s["x"].to(F64), s["w"].to(F64)
        g, u = x @ w[:f].t(), x @ w[f:].t()
        if s["act"] == "silu":
            gate = torch.sigmoid(g)
            slope = gate + g * gate * torch.sigmoid(-g)
        else:
            gate = 0.5 * torch.erfc(-g / math.sqrt(2.0))
            slope = gate + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        act = g * gate
        if kind == "gated":
            return dict(h=act * u)
        dh = s["dy"].to(F64) @ s["down_t"].to(F64).t()
        dg, du = dh * u * slope, dh * act
        return dict(h=act * u, gu=torch.cat([g, u], 1), dgu=torch.cat([dg, du], 1), dx=dg @ w[:f] + du @ w[f:])
    k, n = s["k"], s["n"]
    if s["rows8"]:
        codes, scales = s["q"].to(F32).to(F64), s["scales"].to(F64)
    else:
        codes, scales = _scaled_groups(s["x"].to(F64))
    w = s["w"].to(F32).to(F64)
    y = torch.zeros(s["m"], n, device="cuda", dtype=F64)
    for b in range(_groups(k)):
        columns = slice(b * GROUP, (b + 1) * GROUP)
        part = codes[:, columns] @ w[:, columns].t()
        per_column = s["w_scales"][:, b].to(F64).repeat_interleave(GROUP)[:n]
        y += part * scales[b][:, None] * per_column[None, :]
    if s["residual"] is not None:
        y += s["residual"].to(F64)
    return dict(y=y) if s["rows8"] else dict(y=y, q=codes, scales=scales)
