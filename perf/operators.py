"""The linear-layer operators as they are measured: the matrix product with bias,
activation and residual in its epilogue (``tk.kernels.linear``), the matrix
products grouped by expert with ragged sizes (``tk.kernels.grouped_matmul``),
and the backward pass of each.

``run`` computes an operator in its plain form (elementary torch operations in
32 bits, rounded once at the end), or, where ``own`` is true, through the
framework's kernels on the same buffers.  bf16 operands are rounded N(0, 1)
activations and N(0, 1.2^2 / K) weights, so that pre-activations are of order
one, where an activation bends; e4m3 operands carry a scale per tensor, and
per expert for the experts' weights.
"""

import math
import operator

import torch

own = False

# the framework's largest bf16 product, and the cost that a drawn case may reach
_LARGEST = 8192
_HBM, _TENSOR = 6.5e12, 1.6e15


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _linear(m, n, k, dtype="bf16", act="none", bias=True, residual=False, preact=False):
    return {"op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "preact": preact}


def _linear_backward(m, n, k, act="none", bias=True):
    return {"op": "linear_backward", "m": m, "n": n, "k": k, "act": act, "bias": bias}


def _grouped(e, t, used, n, k, dtype="bf16", act="none", preact=False, skew=0.5):
    return {"op": "grouped", "e": e, "t": t, "used": used, "n": n, "k": k, "dtype": dtype,
            "act": act, "preact": preact, "skew": skew}


def _grouped_backward(e, t, used, n, k, act="none", skew=0.5):
    return {"op": "grouped_backward", "e": e, "t": t, "used": used, "n": n, "k": k, "act": act,
            "skew": skew}


def listed():
    return [
        # serving one sequence: the up projection of one token, bound by the weights' bytes
        dict(_linear(1, 14336, 4096, act="silu"), name="linear decode 1"),
        # serving a batch: the down projection of 16 tokens, back onto the residual stream
        dict(_linear(16, 4096, 14336, residual=True), name="linear decode 16 down"),
        # a short prompt through a narrow layer, every size odd to the tiles
        dict(_linear(777, 1544, 1032, act="gelu_tanh", residual=True, preact=True),
             name="linear ragged 777"),
        # a training step's forward product, keeping what the backward pass needs
        dict(_linear(4096, 4096, 4096, act="gelu", residual=True, preact=True),
             name="linear train 4096"),
        # the largest product, quantised
        dict(_linear(8192, 8192, 8192, dtype="e4m3", act="relu", residual=True),
             name="linear e4m3 8192"),
        # gradients of a small head: latency of the launches counts
        dict(_linear_backward(200, 264, 136, act="silu"), name="linear backward 200"),
        # gradients of a feed-forward layer in training
        dict(_linear_backward(4096, 14336, 4096, act="gelu"), name="linear backward 4096"),
        # serving a mixture of experts: a few tokens, each expert's weights read once
        dict(_grouped(8, 16, 16, 14336, 4096, act="silu"), name="grouped decode 16"),
        # a long prompt over the same experts, sizes skewed as a router leaves them
        dict(_grouped(8, 8192, 8192, 14336, 4096, act="silu"), name="grouped prefill 8192"),
        # many small quantised experts, some without rows, and rows behind the last
        dict(_grouped(64, 4096, 4000, 2048, 1024, dtype="e4m3", skew=1.2), name="grouped e4m3 64"),
        # training the experts
        dict(_grouped_backward(8, 4096, 4096, 4096, 4096, act="silu"),
             name="grouped backward 4096"),
        # training small experts: odd sizes, some experts without rows
        dict(_grouped_backward(32, 1500, 1411, 776, 520, act="gelu_tanh", skew=1.5),
             name="grouped backward odd"),
    ]


def _spread(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, int(round(v / step)) * step)


def _cost(case):
    w = work(case)
    return w["bytes"] / _HBM + w["flops"] / _TENSOR


def draw(rng):
    acts = ["none", "relu", "gelu", "gelu_tanh", "silu"]
    most = {c["op"]: 0.0 for c in listed()}
    for c in listed():
        most[c["op"]] = max(most[c["op"]], _cost(c))
    op = rng.choice(sorted(most))
    while True:
        act = rng.choice(acts)
        n, k = _spread(rng, 128, 14336, 8), _spread(rng, 128, 14336, 8)
        if op == "linear":
            dtype = rng.choice(["bf16", "bf16", "e4m3"])
            if dtype == "e4m3":
                n, k = n // 16 * 16, k // 16 * 16
            case = _linear(_spread(rng, 1, _LARGEST), n, k, dtype, act, rng.random() < 0.7,
                           rng.random() < 0.5, rng.random() < 0.4)
        elif op == "linear_backward":
            case = _linear_backward(_spread(rng, 1, _LARGEST), n, k, act, rng.random() < 0.7)
        else:
            e, t = _spread(rng, 2, 64), _spread(rng, 1, _LARGEST)
            used = max(1, t - rng.choice([0, 0, t // 16, t // 5]))
            skew = rng.choice([0.0, 0.5, 1.0, 1.5])
            if e * n * k > 8 * 14336 * 4096:
                continue
            if op == "grouped":
                dtype = rng.choice(["bf16", "bf16", "e4m3"])
                if dtype == "e4m3":
                    n, k = n // 16 * 16, k // 16 * 16
                case = _grouped(e, t, used, n, k, dtype, act, rng.random() < 0.4, skew)
            else:
                if e * n * k > 8 * 4096 * 4096:
                    continue
                case = _grouped_backward(e, t, used, n, k, act, skew)
        if _cost(case) <= most[op]:
            return case


def work(case):
    """Bytes and operations of one pass: each input read and each output
    written once, each expert that has a row counted once."""
    n, k = case["n"], case["k"]
    if case["op"] in ("linear", "linear_backward"):
        rows, mats = case["m"], 1
    else:
        rows, mats = case["used"], min(case["e"], case["used"])
    el = 1 if case.get("dtype") == "e4m3" else 2
    flops = 2.0 * rows * n * k
    if case["op"] in ("linear", "grouped"):
        b = el * (rows * k + mats * n * k) + 2 * rows * n
        b += 2 * rows * n * (bool(case.get("residual")) + bool(case["preact"]))
        b += 2 * n * bool(case.get("bias"))
        return {"bytes": b, "flops": flops}
    # dout, A, B in; dA, dB out; with an activation the pre-activation in and
    # its gradient out as well
    b = 2 * (rows * n + rows * k + mats * n * k) + 2 * (rows * k) + 2 * case.get("e", 1) * n * k
    b += 4 * rows * n * (case["act"] != "none") + 4 * n * bool(case.get("bias"))
    return {"bytes": b, "flops": 2 * flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _quantised(x):
    scale = float(x.abs().amax()) / 448.0
    return (x / scale).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    """Inputs on the GPU, the group offsets and the output buffers that a
    program keeps between calls."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    def bf16(*shape, std=1.0):
        return normal(*shape, std=std).to(torch.bfloat16)

    def buffer(*shape):
        # what an output holds before the call: the rows behind the last group keep it
        return bf16(*shape) if "e" in case else torch.zeros(*shape, dtype=torch.bfloat16, device="cuda")

    n, k = case["n"], case["k"]
    std = 1.2 / math.sqrt(k)
    s = dict(case)
    if "e" in case:
        e, rows = case["e"], case["t"]
        # how many rows a router gives each expert: popularity ~ rank^-skew, the
        # ranks in an order of their own, so that thin experts get none
        pop = (torch.arange(1, e + 1, device="cuda", dtype=torch.float32)) ** -case["skew"]
        pop = pop[torch.randperm(e, generator=g, device="cuda")]
        to = torch.multinomial(pop, case["used"], replacement=True, generator=g)
        counts = torch.bincount(to, minlength=e)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["most"] = int(counts.max())
        b_shape = (e, k, n)
    else:
        rows, b_shape = case["m"], (k, n)
    if case.get("dtype") == "e4m3":
        s["A"], s["scale_a"] = _quantised(normal(rows, k))
        if "e" in case:
            w = normal(*b_shape, std=std) * (0.5 + torch.rand(e, 1, 1, generator=g, device="cuda"))
            s["scale_b"] = w.abs().amax((1, 2)) / 448.0
            s["B"] = (w / s["scale_b"][:, None, None]).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
        else:
            s["B"], s["scale_b"] = _quantised(normal(*b_shape, std=std))
    else:
        s["A"], s["B"] = bf16(rows, k), bf16(*b_shape, std=std)
    if case["op"] in ("linear", "grouped"):
        s["out"] = buffer(rows, n)
        s["pre"] = buffer(rows, n) if case["preact"] else None
        s["b"] = bf16(n, std=0.5) if case.get("bias") else None
        s["res"] = bf16(rows, n) if case.get("residual") else None
    else:
        s["dout"] = bf16(rows, n, std=1.0 / 64)
        bent = case["act"] != "none"
        s["z"] = bf16(rows, n, std=1.2) if bent else None
        s["dz"] = buffer(rows, n) if bent else None
        s["dA"] = buffer(rows, k)
        s["dB"] = torch.zeros(*b_shape, dtype=torch.bfloat16, device="cuda")
        s["db"] = torch.zeros(n, dtype=torch.float32, device="cuda") if case.get("bias") else None
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
_C = math.sqrt(2.0 / math.pi)


def _act(z, name):
    if name == "relu":
        return z.clamp(min=0.0)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(_C * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if name == "gelu_tanh":
        t = torch.tanh(_C * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * _C * (1.0 + 3 * 0.044715 * z * z)
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return p * (1.0 + z * (1.0 - p))
    return torch.ones_like(z)


def _slots(s):
    """Row index of each slot of the groups padded to one length, which slots
    hold a row, and for each row of the buffer its slot and whether it is in a
    group."""
    off = s["offsets"].long()
    lens = off[1:] - off[:-1]
    at = torch.arange(s["most"], device=off.device)
    held = at[None, :] < lens[:, None]
    row = torch.where(held, off[:-1, None] + at[None, :], torch.zeros_like(off[:1]))
    r = torch.arange(s["t"], device=off.device)
    inside = (r >= off[0]) & (r < off[-1])
    grp = (torch.searchsorted(off, r, right=True) - 1).clamp(0, s["e"] - 1)
    slot = torch.where(inside, grp * s["most"] + (r - off[grp]), torch.zeros_like(r))
    return row, held, slot, inside


def _pad(x, row, held):
    return torch.where(held[:, :, None], x[row], torch.zeros((), dtype=x.dtype, device=x.device))


def _plain_linear(s):
    z = s["A"].float() @ s["B"].float()
    if s["dtype"] == "e4m3":
        z = z * (s["scale_a"] * s["scale_b"])
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, s["act"])
    if s["res"] is not None:
        y = y + s["res"].float()
    got = {"out": y.to(torch.bfloat16)}
    if s["preact"]:
        got["pre"] = z.to(torch.bfloat16)
    return got


def _plain_linear_backward(s):
    dz = s["dout"].float()
    if s["act"] != "none":
        dz = dz * _act_slope(s["z"].float(), s["act"])
    got = {"dA": (dz @ s["B"].float().t()).to(torch.bfloat16),
           "dB": (s["A"].float().t() @ dz).to(torch.bfloat16)}
    if s["bias"]:
        got["db"] = dz.sum(0)
    if s["act"] != "none":
        got["dz"] = dz.to(torch.bfloat16)
    return got


def _plain_grouped(s):
    row, held, slot, inside = _slots(s)
    a, b = _pad(s["A"].float(), row, held), s["B"].float()
    z = torch.bmm(a, b)
    if s["dtype"] == "e4m3":
        z = z * (s["scale_a"] * s["scale_b"])[:, None, None]
    z = z.reshape(-1, s["n"])[slot]
    y = _act(z, s["act"]).to(torch.bfloat16)
    got = {"out": torch.where(inside[:, None], y, s["out"])}
    if s["preact"]:
        got["pre"] = torch.where(inside[:, None], z.to(torch.bfloat16), s["pre"])
    return got


def _plain_grouped_backward(s):
    row, held, slot, inside = _slots(s)
    dz = s["dout"].float()
    if s["act"] != "none":
        dz = dz * _act_slope(s["z"].float(), s["act"])
    padded = _pad(dz, row, held)
    da = torch.bmm(padded, s["B"].float().transpose(1, 2)).reshape(-1, s["k"])[slot]
    db = torch.bmm(_pad(s["A"].float(), row, held).transpose(1, 2), padded)
    got = {"dA": torch.where(inside[:, None], da.to(torch.bfloat16), s["dA"]),
           "dB": db.to(torch.bfloat16)}
    if s["act"] != "none":
        got["dz"] = torch.where(inside[:, None], dz.to(torch.bfloat16), s["dz"])
    return got


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
# what of a state is wrapped for the framework's call
_BUFFERS = ("A", "B", "b", "res", "out", "pre", "offsets", "scale_b", "dout", "z", "dz", "dA", "dB", "db")


def _own_call(s):
    """The operator's handle and the arguments that a program keeps for it:
    device arrays over the state's buffers."""
    import numpy as np

    import thork_b200 as tk

    rt = tk.runtime

    def arr(t):
        if t is None:
            return None
        as_np = {torch.bfloat16: np.uint16, torch.float8_e4m3fn: np.uint8,
                 torch.float32: np.float32, torch.int32: np.int32}[t.dtype]
        return rt.wrap_pointer(t.data_ptr(), tuple(t.shape), as_np, owner=t)

    act = s["act"]
    dtype = tk.dt.float8_e4m3 if s.get("dtype") == "e4m3" else tk.dt.bfloat16
    a, b = arr(s["A"]), arr(s["B"])
    if s["op"] == "linear":
        f = tk.kernels.linear(s["m"], s["n"], s["k"], dtype, activation=act, static_weights=True)
        args = (arr(s["out"]), a, b)
        kw = {"bias": arr(s["b"]), "residual": arr(s["res"]), "preact": arr(s["pre"])}
        if s["dtype"] == "e4m3":
            kw.update(scale_a=s["scale_a"], scale_b=s["scale_b"])
        got = {"out": s["out"]}
        if s["preact"]:
            got["pre"] = s["pre"]
    elif s["op"] == "linear_backward":
        f = tk.kernels.linear_backward(s["m"], s["n"], s["k"], dtype, activation=act)
        args = (arr(s["dA"]), arr(s["dB"]), arr(s["db"]), arr(s["dout"]), a, b)
        kw = {"preact": arr(s["z"]), "dpre": arr(s["dz"])}
        got = {"dA": s["dA"], "dB": s["dB"]}
        if s["bias"]:
            got["db"] = s["db"]
        if act != "none":
            got["dz"] = s["dz"]
    elif s["op"] == "grouped":
        f = tk.kernels.grouped_matmul(s["e"], s["t"], s["n"], s["k"], dtype, activation=act,
                                      static_weights=True)
        args = (arr(s["out"]), a, b, arr(s["offsets"]))
        kw = {"preact": arr(s["pre"])}
        if s["dtype"] == "e4m3":
            kw.update(scale_a=s["scale_a"], scale_b=arr(s["scale_b"]))
        got = {"out": s["out"]}
        if s["preact"]:
            got["pre"] = s["pre"]
    else:
        f = tk.kernels.grouped_matmul_backward(s["e"], s["t"], s["n"], s["k"], dtype, activation=act)
        args = (arr(s["dA"]), arr(s["dB"]), arr(s["dout"]), a, b, arr(s["offsets"]))
        kw = {"preact": arr(s["z"]), "dpre": arr(s["dz"])}
        got = {"dA": s["dA"], "dB": s["dB"]}
        if act != "none":
            got["dz"] = s["dz"]
    return f, args, kw, got


def _own(s):
    """The framework's call on torch's current stream; the wraps are made anew
    for a state whose buffers are others than at the call before."""
    kept = s.get("call")
    if kept is None or any(map(operator.is_not, kept["pick"](s), kept["buffers"])):
        pick = operator.itemgetter(*(name for name in _BUFFERS if s.get(name) is not None))
        kept = s["call"] = {"pick": pick, "buffers": pick(s), "call": _own_call(s), "handle": -1}
    # torch.cuda.current_stream().cuda_stream without the Stream object, which
    # takes longer to make than the rest of this function
    handle = torch._C._cuda_getCurrentRawStream(kept["buffers"][0].device.index)
    if handle != kept["handle"]:
        from thork_b200 import runtime

        kept["handle"], kept["stream"] = handle, runtime.Stream.from_handle(handle)
    f, args, kw, got = kept["call"]
    f(*args, **kw, stream=kept["stream"], sync=False)
    return got


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "linear_backward": _plain_linear_backward,
            "grouped": _plain_grouped, "grouped_backward": _plain_grouped_backward}[state["op"]](state)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_act(z, name):
    """(value, slope) of the activation at z."""
    if name == "relu":
        pos = (z > 0).double()
        return z * pos, pos
    if name == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        u = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        p = torch.sigmoid(2 * u)  # (1 + tanh u) / 2
        return z * p, p + z * 2 * p * (1 - p) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    return z, torch.ones_like(z)


def exact(case, seed):
    s = prepare(case, seed)
    if "e" in case:
        off = s["offsets"].tolist()
        groups = [(off[i], off[i + 1], s["B"][i]) for i in range(case["e"])]
    else:
        groups = [(0, case["m"], s["B"])]
    if case["op"] in ("linear", "grouped"):
        out = s["out"].double()
        pre = s["pre"].double() if case["preact"] else None
        for i, (lo, hi, b) in enumerate(groups):
            z = torch.matmul(s["A"][lo:hi].double(), b.double())
            if case["dtype"] == "e4m3":
                sb = s["scale_b"]
                z *= s["scale_a"] * (float(sb[i]) if "e" in case else sb)
            if s["b"] is not None:
                z += s["b"].double()
            if pre is not None:
                pre[lo:hi] = z
            out[lo:hi] = _exact_act(z, case["act"])[0]
            if s["res"] is not None:
                out[lo:hi] += s["res"][lo:hi].double()
        return {"out": out, "pre": pre} if pre is not None else {"out": out}
    da, db = s["dA"].double(), s["dB"].double()
    dz = s["dz"].double() if case["act"] != "none" else None
    for i, (lo, hi, b) in enumerate(groups):
        g = s["dout"][lo:hi].double()
        if dz is not None:
            g = g * _exact_act(s["z"][lo:hi].double(), case["act"])[1]
            dz[lo:hi] = g
        da[lo:hi] = torch.matmul(g, b.double().t())
        grad = torch.matmul(s["A"][lo:hi].double().t(), g)
        if "e" in case:
            db[i] = grad
        else:
            db = grad
        if s["db"] is not None:
            s["db"] = g.sum(0)
    got = {"dA": da, "dB": db}
    if s["db"] is not None:
        got["db"] = s["db"]
    if dz is not None:
        got["dz"] = dz
    return got
