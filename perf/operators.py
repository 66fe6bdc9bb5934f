"""The 8-bit operators, as calls to be measured: what each call has in hand, its plain form, and its exact answer.

    linear     Y[m, n] = s_A[m] * s_B[n] * sum_k A[m, k] * Bt[n, k] (+ bias[n]): a product of 8-bit integers, a scale for
               each token (row of A) and each channel (row of Bt), the result in bf16, fp16 or fp32
    quantise   s[m] = max_k |x[m, k]| / 127, q[m, k] = x[m, k] / s[m] rounded half to even: what gives `linear` its operands
    norm       h = x + r rounded to x's type (r may be absent), t = h * w, s[m] = max_k |t| / 127 / sqrt(mean_k(h^2) + eps)
               and q = 127 * t / max_k |t| rounded half to even: the root-mean-square norm before `linear`, in one pass

q is whole numbers and has to be equal: it is computed where rounding cannot move a value across a border (64 bits here).
The rounding of h to x's type and of t to 32 bits belong to the definition: h is what the residual stream holds.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


def linear(name, m, n, k, dtype="bf16", bias=False, pad=0):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias, "pad": pad}


def rows(name, op, m, k, dtype="bf16", residual=False, pad=0):
    return {"name": name, "op": op, "m": m, "k": k, "dtype": dtype, "residual": residual, "pad": pad}


def listed():
    return [
        # generation, one sequence: the weights are read once for one token, latency is all there is
        linear("linear 1x4096x4096", 1, 4096, 4096),
        # generation, a batch of sequences: still bound by the weights
        linear("linear 32x8192x8192", 32, 8192, 8192),
        # nothing even: 77 tokens, a projection with a bias, rows further apart than they are long
        linear("linear 77x1003x1111 odd", 77, 1003, 1111, "fp32", bias=True, pad=48),
        # a short prompt
        linear("linear 512x4096x4096", 512, 4096, 4096, "fp16"),
        # three of the shapes that the fp16 product is measured on: a small one, one with a short K, a large one
        linear("linear 2048x2048x2048", 2048, 2048, 2048),
        linear("linear 4096x4096x1024", 4096, 4096, 1024, "fp32"),
        linear("linear 8192x8192x8192", 8192, 8192, 8192),
        # activations of a few tokens, odd length
        rows("quantise 5x1111 odd", "quantise", 5, 1111),
        # a weight matrix on its way into 8 bits
        rows("quantise 8192x8192 fp32", "quantise", 8192, 8192, "fp32"),
        # the norm before a projection: one token, a ragged batch without a residual, a long prompt
        rows("norm 1x4096", "norm", 1, 4096, residual=True),
        rows("norm 333x5121 odd", "norm", 333, 5121, "fp16", pad=15),
        rows("norm 16384x4096", "norm", 16384, 4096, residual=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high):
    """Spread over the logarithm; two in five as drawn (mostly odd), the others multiples of 64 or 16."""
    v, how = _log(rng, low, high), rng.random()
    step = 1 if how < 0.4 else 64 if how < 0.8 else 16
    return max(low, min(high, (v + step // 2) // step * step))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if rng.random() < 0.55:
        while True:
            m = _size(rng, 1, 64) if rng.random() < 0.4 else _size(rng, 1, 8192)
            n, k = _size(rng, 48, 16384), _size(rng, 48, 16384)
            if m * n * k <= 8192 ** 3 and n * k <= 1 << 27:
                break
        c = linear("", max(1, m), n, k, dtype, rng.random() < 0.3, rng.choice([0, 0, 16, 80]))
    else:
        op = rng.choice(["quantise", "norm"])
        while True:
            m, k = _size(rng, 1, 16384), _size(rng, 48, 16384)
            if m * k * SIZE[dtype] <= 1 << 27:
                break
        c = rows("", op, max(1, m), k, dtype, op == "norm" and rng.random() < 0.6, rng.choice([0, 0, 1, 16]))
    del c["name"]
    return c


def _strided(m, k, ld, make):
    """m rows of k values, ld apart: a view of a wider matrix whose other columns hold values too."""
    return make(m, ld)[:, :k]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    m, k, kind = case["m"], case["k"], TYPES[case["dtype"]]
    ld = -(-k // 16) * 16 + case["pad"]  # rows of 8-bit operands start on 16-byte boundaries
    if case["op"] == "linear":
        n = case["n"]

        def integers(r, c):  # what quantised activations and weights look like: normal, the largest of a row near 127
            return (torch.randn(r, c, generator=g, device="cuda") * 36).round_().clamp_(-127, 127).to(torch.int8)

        def scales(r, around):
            return around * torch.exp(0.5 * torch.randn(r, generator=g, device="cuda"))

        s = {"op": "linear", "m": m, "a": _strided(m, k, ld, integers), "sa": scales(m, 0.02), "b": _strided(n, k, ld, integers),
             "sb": scales(n, 0.001), "kind": kind, "ld": ld, "bias": torch.randn(n, generator=g, device="cuda") if case["bias"] else None}
        s["y"] = torch.empty(m, n, dtype=kind, device="cuda")
        if own:  # a program keeps a plan for each weight matrix
            import warpc_public_release_b200 as w
            s["plan"] = w.Int8Plan(n, k, s["b"].data_ptr(), s["sb"].data_ptr(), dBias=s["bias"].data_ptr() if case["bias"] else None,
                                   out=case["dtype"], ldb=ld)
        return s

    def activations(r, c):  # a spread of row magnitudes, and a few channels far larger than the others
        x = torch.randn(r, c, generator=g, device="cuda")
        x *= torch.exp(torch.randn(r, 1, generator=g, device="cuda"))
        x[:, torch.randperm(c, generator=g, device="cuda")[: max(1, c // 256)]] *= 20
        return x.to(kind)

    wide = k + case["pad"]
    s = {"op": case["op"], "m": m, "k": k, "dtype": case["dtype"], "x": _strided(m, k, wide, activations), "ldx": wide, "ldq": ld,
         "q": torch.zeros(m, ld, dtype=torch.int8, device="cuda"), "scale": torch.empty(m, device="cuda"), "r": None, "h": None}
    if case["op"] == "norm":
        s["w"] = (1 + 0.3 * torch.randn(k, generator=g, device="cuda")).to(kind)
        if case["residual"]:
            s["r"] = _strided(m, k, wide, activations)
            s["h"] = torch.empty(m, k, dtype=kind, device="cuda")
    return s


def _plain_quantise(t):
    """t in 32 bits -> 8 bits and the largest value of each row; the quotient in 64 bits, where no value next to a border moves."""
    top = t.abs().amax(1, keepdim=True)
    q = torch.round(t.double() * 127 / top.double())
    return torch.where(top > 0, q, 0.0).to(torch.int8), top[:, 0]


def _run_plain(s):
    if s["op"] == "linear":
        y = (s["a"].float() @ s["b"].float().t()) * s["sa"][:, None] * s["sb"]
        if s["bias"] is not None:
            y = y + s["bias"]
        return y.to(s["kind"])
    if s["op"] == "quantise":
        q, top = _plain_quantise(s["x"].float())
        return {"q": q, "scale": top / 127}
    h = s["x"].float()
    if s["r"] is not None:
        h = (h + s["r"].float()).to(s["x"].dtype).float()
    q, top = _plain_quantise(h * s["w"].float())
    out = {"q": q, "scale": top / 127 / torch.sqrt((h * h).mean(1) + EPS)}
    if s["r"] is not None:
        out["h"] = h.to(s["x"].dtype)
    return out


def _run_own(s):
    import warpc_public_release_b200 as w
    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "linear":
        s["plan"].launch(s["m"], s["a"].data_ptr(), s["sa"].data_ptr(), s["y"].data_ptr(), lda=s["ld"], stream=stream)
        return s["y"]
    out = {"q": s["q"][:, : s["k"]], "scale": s["scale"]}
    if s["op"] == "quantise":
        w.quantise_rows(s["m"], s["k"], s["x"].data_ptr(), s["q"].data_ptr(), s["scale"].data_ptr(), dtype=s["dtype"], ldx=s["ldx"],
                        ldq=s["ldq"], stream=stream)
        return out
    more = {}
    if s["r"] is not None:
        more = {"dR": s["r"].data_ptr(), "ldr": s["ldx"], "dH": s["h"].data_ptr()}
        out["h"] = s["h"]
    w.norm_quantise_rows(s["m"], s["k"], s["x"].data_ptr(), s["w"].data_ptr(), EPS, s["q"].data_ptr(), s["scale"].data_ptr(), dtype=s["dtype"],
                         ldx=s["ldx"], ldq=s["ldq"], stream=stream, **more)
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    m, k, size = case["m"], case["k"], SIZE[case["dtype"]]
    if case["op"] == "linear":
        n = case["n"]
        return {"bytes": m * k + n * k + m * n * size + 4 * (m + n + (n if case["bias"] else 0)), "flops": 2 * m * n * k}
    moved = m * k * (size + 1) + 4 * m
    if case["op"] == "norm":
        moved += k * size + (2 * m * k * size if case["residual"] else 0)
    return {"bytes": moved, "flops": (7 if case["op"] == "norm" else 3) * m * k}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "linear":
        y = torch.einsum("mk,nk->mn", s["a"].double(), s["b"].double())  # whole numbers below 2^53: exact
        y.mul_(torch.outer(s["sa"].double(), s["sb"].double()))
        return y if s["bias"] is None else y.add_(s["bias"].double().expand_as(y))
    x = s["x"].double()
    if s["op"] == "quantise":
        return {"q": None, "scale": torch.linalg.vector_norm(x, ord=math.inf, dim=1) / 127}
    total = x if s["r"] is None else x + s["r"].double()
    h = total.to(s["x"].dtype).double()  # the sum as the residual stream holds it
    size = torch.linalg.vector_norm(h, dim=1) / math.sqrt(case["k"])
    top = torch.linalg.vector_norm(h * s["w"].double(), ord=math.inf, dim=1)
    out = {"q": None, "scale": top / (127 * torch.sqrt(size * size + EPS))}
    return out if s["r"] is None else {**out, "h": total}
