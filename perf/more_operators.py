"""What every token of a mixture-of-experts layer passes through beside the routed experts, as cases that can be timed one by one.

Three families:

  norm  the root-mean-square norm with the residual's addition, its output in 16 bits and, with "quantize", as FP8 codes with a scale for
        each 128 values, as dispatch takes them; with "backward" also the gradients of its input and its weight
  ffn   the gated feed-forward block of a shared expert or a dense layer: gate and up products, SwiGLU, down product; with "backward"
        also the gradients of its input and its matrices
  w8    a product in 8-bit integers with scales of tokens and channels: of rows in 16 bits that the call quantises, of codes, or of what
        a norm in front of it leaves in 8 bits ("norm", with the residual's addition)

`own` says whose code computes them: this package's kernels, or (False) elementary torch operations in 32 bits, which run on a tree
that lacks the kernels.  Sizes are those of this repository's benchmark, presets and tests, and generic ones beside them.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6

# Upper bounds of a drawn case, so that none costs more than the largest listed one.
_MOST_NORM = 16384 * 7168
_MOST_FFN = 8192 * 2048 * 7168
_MOST_W8 = 8192 * 4096 * 7168


def listed():
    return [
        # The norm of one decoded token in front of a layer whose dispatch takes FP8: launch and host time only.
        dict(name="norm 1x7168 fp8", family="norm", tokens=1, hidden=7168, dtype="bf16", weight="bf16", residual=True, quantize="fp8",
             backward=False),
        # A prefill chunk on its way into an FP8 dispatch, with the residual stream's update.
        dict(name="norm 4096x7168 fp8", family="norm", tokens=4096, hidden=7168, dtype="bf16", weight="bf16", residual=True, quantize="fp8",
             backward=False),
        # A fine-tuning batch in half precision, sizes that are no powers of two; no residual in front of the first layer.
        dict(name="norm train 777x2880 fp16", family="norm", tokens=777, hidden=2880, dtype="fp16", weight="fp32", residual=False,
             quantize="", backward=True),
        # The largest: a training batch, both directions, the stream's own gradient added on the way back.
        dict(name="norm train 16384x7168", family="norm", tokens=16384, hidden=7168, dtype="bf16", weight="fp32", residual=True, quantize="",
             backward=True),
        # One decoded token through a shared expert: nothing but the stream of its weights.
        dict(name="ffn 1x7168x2048", family="ffn", tokens=1, hidden=7168, inter=2048, dtype="bf16", backward=False),
        # A speculative batch of a smaller model, sizes that are no whole tiles.
        dict(name="ffn 33x2880x1408 fp16", family="ffn", tokens=33, hidden=2880, inter=1408, dtype="fp16", backward=False),
        # A prefill chunk: too many tokens for a stream of weights, few for the matrix cores.
        dict(name="ffn 512x7168x2048", family="ffn", tokens=512, hidden=7168, inter=2048, dtype="bf16", backward=False),
        # A small training batch with a ragged number of tokens.
        dict(name="ffn train 1000x2880x1408", family="ffn", tokens=1000, hidden=2880, inter=1408, dtype="bf16", backward=True),
        # The largest: a training batch through the shared expert, both directions.
        dict(name="ffn train 8192x7168x2048", family="ffn", tokens=8192, hidden=7168, inter=2048, dtype="bf16", backward=True),
        # One decoded token: norm, then the shared expert's gate and up matrices in 8 bits.
        dict(name="w8 norm 1x7168 to 4096", family="w8", tokens=1, inputs=7168, outputs=4096, dtype="bf16", rows="norm"),
        # A decode batch whose rows are quantised in the call, an odd number of channels.
        dict(name="w8 100x2880 to 1407 fp16", family="w8", tokens=100, inputs=2880, outputs=1407, dtype="fp16", rows="wide"),
        # The largest: a prefill batch that a norm left in codes, through the gate and up matrices.
        dict(name="w8 8192x7168 to 4096", family="w8", tokens=8192, inputs=7168, outputs=4096, dtype="bf16", rows="codes"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _multiple(rng, step, low, high):
    return _log_int(rng, -(-low // step), high // step) * step


def draw(rng):
    family = rng.choices(("norm", "ffn", "w8"), weights=(4, 5, 3))[0]
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    while True:
        if family == "norm":
            case = dict(family=family, tokens=_log_int(rng, 1, 32768), hidden=_multiple(rng, 16, 256, 16384), dtype=dtype,
                        weight=rng.choice((dtype, "fp32")), residual=rng.random() < 0.7, quantize=rng.choice(("", "", "fp8")),
                        backward=rng.random() < 0.5)
            if case["tokens"] * case["hidden"] <= _MOST_NORM:
                return case
        elif family == "ffn":
            case = dict(family=family, tokens=_log_int(rng, 1, 16384), hidden=_multiple(rng, 8, 256, 8192), inter=_multiple(rng, 8, 128, 8192),
                        dtype=dtype, backward=rng.random() < 0.5)
            if max(case["tokens"], 1024) * case["hidden"] * case["inter"] <= _MOST_FFN:
                return case
        else:
            case = dict(family=family, tokens=_log_int(rng, 1, 16384), inputs=_multiple(rng, 16, 256, 16384), outputs=_log_int(rng, 64, 16384),
                        dtype=dtype, rows=rng.choice(("wide", "codes", "norm")))
            if max(case["tokens"], 1024) * case["inputs"] * case["outputs"] <= _MOST_W8:
                return case


# ---- inputs ------------------------------------------------------------------------------------------------------------------
_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _normal(gen, *shape, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda") * scale


def _stream(case, gen, hidden):
    """Rows of a residual stream: tokens of uneven size, a few columns that are much larger than the others."""
    size = 0.5 + torch.rand((case["tokens"], 1), generator=gen, device="cuda")
    columns = torch.ones((hidden,), device="cuda")
    columns[torch.randperm(hidden, generator=gen, device="cuda")[: max(1, hidden // 512)]] = 12.0
    return (_normal(gen, case["tokens"], hidden) * size * columns).to(_DTYPES[case["dtype"]])


class _State:
    def __init__(self, case, **fields):
        self.case = case
        self.__dict__.update(fields)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, tokens = _DTYPES[case["dtype"]], case["tokens"]
    if case["family"] == "norm":
        hidden = case["hidden"]
        training = case["backward"]
        return _State(
            case, x=_stream(case, gen, hidden), residual=_stream(case, gen, hidden) if case["residual"] else None,
            weight=(1.0 + _normal(gen, hidden, scale=0.2)).to(_DTYPES[case["weight"]]),
            grad_y=_normal(gen, tokens, hidden, scale=0.01).to(dtype) if training else None,
            grad_stream=_normal(gen, tokens, hidden, scale=0.01).to(dtype) if training and case["residual"] else None)
    if case["family"] == "ffn":
        hidden, inter = case["hidden"], case["inter"]
        return _State(
            case, x=_normal(gen, tokens, hidden).to(dtype), gate_up=_normal(gen, 2 * inter, hidden, scale=hidden**-0.5).to(dtype),
            down=_normal(gen, hidden, inter, scale=inter**-0.5).to(dtype),
            grad_y=_normal(gen, tokens, hidden, scale=0.1).to(dtype) if case["backward"] else None)
    inputs, outputs = case["inputs"], case["outputs"]
    state = _State(
        case, codes=(_normal(gen, outputs, inputs, scale=32.0)).round_().clamp_(-127, 127).to(torch.int8),
        scales=inputs**-0.5 / 32.0 * (0.7 + 0.6 * torch.rand((outputs,), generator=gen, device="cuda")))
    if case["rows"] == "codes":
        state.x_codes = _normal(gen, tokens, inputs, scale=32.0).round_().clamp_(-127, 127).to(torch.int8)
        state.x_scales = (0.5 + torch.rand((tokens,), generator=gen, device="cuda")) / 32.0
        return state
    state.x = _stream(case, gen, inputs)
    if case["rows"] == "norm":
        state.residual, state.weight = _stream(case, gen, inputs), (1.0 + _normal(gen, inputs, scale=0.2)).to(dtype)
    return state


# ---- the package's operators ---------------------------------------------------------------------------------------------------
def _run_own(state):
    from deepep_amd import dense, w8

    case = state.case
    if case["family"] == "norm":
        out = dense.rms_norm(state.x, state.weight, state.residual, eps=EPS, quantize=case["quantize"] or None)
        got = [out.y, out.rstd]
        if case["residual"]:
            got.append(out.stream)
        if case["quantize"]:
            got += [out.codes, out.scales]
        if case["backward"]:
            got += dense.rms_norm_backward(state.grad_y, out.stream, state.weight, out.rstd, state.grad_stream)
        return got
    if case["family"] == "ffn":
        if not case["backward"]:
            return [dense.gated_ffn(state.x, state.gate_up, state.down)]
        y, kept = dense.gated_ffn(state.x, state.gate_up, state.down, keep=True)
        return [y, *dense.gated_ffn_backward(state.grad_y, state.x, state.gate_up, state.down, kept)]
    weights = w8.W8Weights(state.codes, state.scales)
    dtype = _DTYPES[case["dtype"]]
    if case["rows"] == "codes":
        return [w8.matmul((state.x_codes, state.x_scales), weights, dtype=dtype)]
    if case["rows"] == "wide":
        return [w8.matmul(state.x, weights)]
    out = dense.rms_norm(state.x, state.weight, state.residual, eps=EPS, quantize="int8", output=False)
    return [out.stream, w8.matmul((out.codes, out.scales), weights, dtype=dtype)]


# ---- the same in elementary operations, 32 bits ----------------------------------------------------------------------------------
def _plain_norm(state):
    """(the stream in its type and in 32 bits, 1 / root mean square, the normed rows in 32 bits)."""
    stream = state.x
    if state.residual is not None:
        stream = (state.x.to(torch.float32) + state.residual.to(torch.float32)).to(state.x.dtype)
    s = stream.to(torch.float32)
    rstd = 1.0 / torch.sqrt((s * s).mean(dim=1) + EPS)
    return stream, s, rstd, s * rstd[:, None] * state.weight.to(torch.float32)


def _plain_blocks(v):
    """FP8 codes of blocks of 128 values and the blocks' scales; a short last block is filled up with zeros."""
    tokens, hidden = v.shape
    blocks = -(-hidden // 128)
    padded = torch.zeros((tokens, blocks * 128), device=v.device)
    padded[:, :hidden] = v
    padded = padded.view(tokens, blocks, 128)
    largest = padded.abs().amax(dim=2).clamp_min(1e-4)
    codes = (padded * (448.0 / largest)[:, :, None]).view(tokens, -1)[:, :hidden].to(torch.float8_e4m3fn)
    return codes.contiguous(), largest / 448.0


def _plain_tokens(v):
    """8-bit integer codes (as 32-bit numbers) and scales of the tokens."""
    largest = v.abs().amax(dim=1).clamp_min(1e-20)
    return torch.round(v * (127.0 / largest)[:, None]).clamp(-127.0, 127.0), largest / 127.0


def _run_plain(state):
    case = state.case
    dtype = _DTYPES[case["dtype"]]
    if case["family"] == "norm":
        stream, s, rstd, v = _plain_norm(state)
        got = [v.to(dtype), rstd]
        if case["residual"]:
            got.append(stream)
        if case["quantize"]:
            got += _plain_blocks(v)
        if case["backward"]:
            g, hat = state.grad_y.to(torch.float32), s * rstd[:, None]
            gw = g * state.weight.to(torch.float32)
            grad = rstd[:, None] * (gw - hat * (gw * hat).mean(dim=1, keepdim=True))
            if state.grad_stream is not None:
                grad = grad + state.grad_stream.to(torch.float32)
            got += [grad.to(dtype), (g * hat).sum(dim=0)]
        return got
    if case["family"] == "ffn":
        x, gate_up, down = (t.to(torch.float32) for t in (state.x, state.gate_up, state.down))
        gate, up = (x @ gate_up.t()).chunk(2, dim=1)
        share = 1.0 / (1.0 + torch.exp(-gate))
        h = gate * share * up
        y = (h @ down.t()).to(dtype)
        if not case["backward"]:
            return [y]
        grad_y = state.grad_y.to(torch.float32)
        grad_h = grad_y @ down
        grad_z = torch.cat([grad_h * up * share * (1.0 + gate * (1.0 - share)), grad_h * gate * share], dim=1)
        return [y, (grad_z @ gate_up).to(dtype), (grad_z.t() @ x).to(dtype), (grad_y.t() @ h).to(dtype)]
    got = []
    if case["rows"] == "codes":
        codes, scales = state.x_codes.to(torch.float32), state.x_scales
    elif case["rows"] == "wide":
        codes, scales = _plain_tokens(state.x.to(torch.float32))
    else:
        stream, _, _, v = _plain_norm(state)
        got.append(stream)
        codes, scales = _plain_tokens(v)
    y = codes @ state.codes.to(torch.float32).t()
    return [*got, (y * scales[:, None] * state.scales).to(dtype)]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------------
def _exact_stream(state):
    """The norm's input: the residual stream as it is held, in the type of its rows."""
    if state.residual is None:
        return state.x.double()
    return (state.x.double() + state.residual.double()).float().to(state.x.dtype).double()


def _exact_normed(s, weight):
    return s / torch.linalg.vector_norm(s, dim=1, keepdim=True).square().div(s.shape[1]).add(EPS).sqrt() * weight.double()


def _exact_tokens(v):
    scale = (v.abs().max(dim=1, keepdim=True).values / 127.0).clamp_min(1e-20 / 127.0)
    return torch.round(v / scale) * scale


def exact(case, seed):
    state = prepare(case, seed)
    if case["family"] == "norm":
        s = _exact_stream(state).requires_grad_(case["backward"])
        weight = state.weight.double().requires_grad_(case["backward"])
        v = _exact_normed(s, weight)
        got = [v.detach(), 1.0 / (s.detach().square().sum(dim=1) / s.shape[1] + EPS).sqrt()]
        if case["residual"]:
            got.append(s.detach())
        if case["quantize"]:
            largest = torch.stack([b.abs().max(dim=1).values for b in v.detach().split(128, dim=1)], dim=1).clamp_min(1e-4)
            # a code stands for this number, before its rounding to 8 bits
            got += [v.detach() * (448.0 / largest).repeat_interleave(128, dim=1)[:, : v.shape[1]], largest / 448.0]
        if case["backward"]:
            grad_s, grad_weight = torch.autograd.grad(v, (s, weight), state.grad_y.double())
            got += [grad_s if state.grad_stream is None else grad_s + state.grad_stream.double(), grad_weight]
        return got
    if case["family"] == "ffn":
        x, gate_up, down = (t.double().requires_grad_(case["backward"]) for t in (state.x, state.gate_up, state.down))
        inter = case["inter"]
        z = torch.matmul(x, gate_up.T)
        y = torch.matmul(torch.sigmoid(z[:, :inter]) * z[:, :inter] * z[:, inter:], down.T)
        if not case["backward"]:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, (x, gate_up, down), state.grad_y.double())]
    matrix = state.codes.double() * state.scales.double()[:, None]
    if case["rows"] == "codes":
        return [(state.x_codes.double() * state.x_scales.double()[:, None]) @ matrix.T]
    if case["rows"] == "wide":
        return [_exact_tokens(state.x.double()) @ matrix.T]
    s = _exact_stream(state)
    return [s, _exact_tokens(_exact_normed(s, state.weight)) @ matrix.T]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------
def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    size, tokens = 2, case["tokens"]
    if case["family"] == "norm":
        cells, weight = tokens * case["hidden"], case["hidden"] * (4 if case["weight"] == "fp32" else 2)
        total = 2 * cells * size + weight + 4 * tokens + (2 * cells * size if case["residual"] else 0)  # x, y; residual, stream
        flops = 5 * cells
        if case["quantize"]:
            total += cells + 4 * tokens * -(-case["hidden"] // 128)
            flops += 3 * cells
        if case["backward"]:  # grad y, grad x, grad weight; the stream's own gradient
            total += 2 * cells * size + 4 * case["hidden"] + (cells * size if case["residual"] else 0)
            flops += 10 * cells
        return {"bytes": total, "flops": flops}
    if case["family"] == "ffn":
        weights = 3 * case["hidden"] * case["inter"]
        rows = 2 * tokens * case["hidden"]
        passes = 3 if case["backward"] else 1
        return {"bytes": ((weights + rows) * (2 if case["backward"] else 1)) * size, "flops": 2 * passes * tokens * weights}
    inputs, outputs = case["inputs"], case["outputs"]
    rows = {"codes": inputs + 4, "wide": inputs * size, "norm": 3 * inputs * size}[case["rows"]]
    return {"bytes": inputs * outputs + 4 * outputs + tokens * (rows + outputs * size), "flops": 2 * tokens * inputs * outputs}
