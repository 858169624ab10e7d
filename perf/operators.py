"""Cases for the 8-bit linear layer's operators: the block-scaled fp8 product, the root-mean-square norm with the
residual's addition and an fp8 output, its backward pass, and the quantisation of a matrix (as it stands and transposed).

An fp8 matrix is [rows][cols] values of e4m3 or e5m2 with one fp32 scale for each block of block_rows x 128 (block_rows 1
for activations and gradients, 128 for weights); a value stands for code * scale."""
import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
FMAX = {"e4m3": 448.0, "e5m2": 57344.0}
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FLOAT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
TINY = 2.0 ** -126          # smallest scale: a block of zeros has it


def listed():
    return [
        # product, one token against a square projection: the latency of a decoding step
        dict(name="gemm 1 token", op="gemm", m=1, n=4096, k=4096, a="e4m3", b="e4m3", b_rows=128, d="bf16", add=False),
        # product, a decoding batch against a wide projection: the weights' bytes count
        dict(name="gemm 48 tokens", op="gemm", m=48, n=4096, k=8192, a="e4m3", b="e4m3", b_rows=128, d="bf16", add=False),
        # product, a ragged prefill: no size a multiple of a tile, the last block of 128 cut
        dict(name="gemm ragged", op="gemm", m=777, n=1111, k=2008, a="e4m3", b="e4m3", b_rows=128, d="f16", add=False),
        # product, ordinary training forward at this repository's second configuration
        dict(name="gemm 8192x4096x2048", op="gemm", m=8192, n=4096, k=2048, a="e4m3", b="e4m3", b_rows=128, d="bf16", add=False),
        # product, weight gradient: both operands scaled by row over tokens, gradients in e5m2, added to the fp32 gradient
        dict(name="gemm weight gradient", op="gemm", m=4096, n=4096, k=8192, a="e5m2", b="e4m3", b_rows=1, d="f32", add=True),
        # product, the largest: a long prefill through a feed-forward projection
        dict(name="gemm 16384x4096x8192", op="gemm", m=16384, n=4096, k=8192, a="e4m3", b="e4m3", b_rows=128, d="bf16", add=False),
        # norm, one token of a decoding step
        dict(name="norm 1 token", op="norm", rows=1, cols=4096, t="bf16", res=True, y=False, q="e4m3"),
        # norm, a training batch that keeps the sum and the plain output for the backward pass
        dict(name="norm 8192x4096", op="norm", rows=8192, cols=4096, t="bf16", res=True, y=True, q="e4m3"),
        # the norm's backward, few rows of an odd count
        dict(name="norm backward 61x5120", op="normb", rows=61, cols=5120, t="bf16", res=True),
        # the norm's backward, a training batch
        dict(name="norm backward 8192x4096", op="normb", rows=8192, cols=4096, t="bf16", res=True),
        # quantisation, weights in fp32 once per optimiser step: 128 x 128 blocks, powers of two, both orientations
        dict(name="quantise weights", op="quant", rows=1000, cols=1500, t="f32", q="e4m3", block=128, rule="pow2", both=True),
        # quantisation, gradients of a training batch by row for the input's gradient and by column for the weights'
        dict(name="quantise 8192x4096", op="quant", rows=8192, cols=4096, t="bf16", q="e5m2", block=1, rule="amax", both=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "gemm", "norm", "normb", "quant"])
    if op == "gemm":
        while True:
            m = _log(rng, 1, 64) if rng.random() < 0.4 else _log(rng, 65, 16384)
            n, k = _log(rng, 64, 16384), _log(rng, 64, 16384)
            if rng.random() < 0.4:          # most real projections are multiples of 128
                n, k = -(-n // 128) * 128, -(-k // 128) * 128
            if m * n * k <= 2 ** 39 and m * n <= 2 ** 26:
                break
        return dict(op=op, m=m, n=n, k=k, a=rng.choice(["e4m3", "e4m3", "e5m2"]), b="e4m3", b_rows=rng.choice([128, 128, 1]),
                    d=rng.choice(["bf16", "f16", "f32"]), add=rng.random() < 0.25)
    while True:
        rows, cols = _log(rng, 1, 16384), _log(rng, 64, 16384)
        if rng.random() < 0.5:
            cols = -(-cols // 128) * 128
        if rows * cols <= 2 ** 25:
            break
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        y = rng.random() < 0.5
        return dict(op=op, rows=rows, cols=cols, t=t, res=rng.random() < 0.7, y=y, q=rng.choice(["e4m3", "e5m2"]))
    if op == "normb":
        return dict(op=op, rows=rows, cols=cols, t=t, res=rng.random() < 0.7)
    return dict(op=op, rows=rows, cols=cols, t=t, q=rng.choice(["e4m3", "e5m2"]), block=rng.choice([1, 128]),
                rule=rng.choice(["amax", "pow2"]), both=rng.random() < 0.7)


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _activations(g, rows, cols):
    """Normal values, some channels ten times larger than the rest (as hidden states have them), the last of many rows
    zero (a padded token)."""
    x = torch.randn(rows, cols, device=DEV, generator=g)
    x *= 1.0 + 9.0 * (torch.rand(cols, device=DEV, generator=g) < 0.01).float()
    if rows > 8:
        x[-1] = 0.0
    return x


def _blocks(x, block_rows, fill=0.0):
    """x [rows][cols] as [row blocks][block_rows][column blocks][128], the edges filled."""
    rows, cols = x.shape
    r, c = -(-rows // block_rows), -(-cols // 128)
    p = torch.full((r * block_rows, c * 128), fill, dtype=x.dtype, device=x.device)
    p[:rows, :cols] = x
    return p.view(r, block_rows, c, 128)


def _quantised(x, kind, block_rows, pitch=16):
    """An fp8 matrix in hand before the call: codes with a row pitch that is a multiple of 16, scales by block."""
    rows, cols = x.shape
    s = (_blocks(x, block_rows).abs().amax((1, 3)) / FMAX[kind]).clamp_min(TINY)
    code = torch.zeros(rows, -(-cols // pitch) * pitch, device=DEV, dtype=FP8[kind])[:, :cols]
    code.copy_((x / _spread(s, block_rows, rows, cols)).to(FP8[kind]))
    if block_rows == 1:
        s = s.t().contiguous().t()          # row scales of one block of columns lie together
    return code, s


def _spread(s, block_rows, rows, cols):
    return s.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def _empty_fp8(rows, cols, kind, block_rows):
    code = torch.empty(rows, -(-cols // 16) * 16, device=DEV, dtype=FP8[kind])[:, :cols]
    if block_rows == 1:
        return code, torch.empty(-(-cols // 128), rows, device=DEV).t()
    return code, torch.empty(-(-rows // 128), -(-cols // 128), device=DEV)


_context = None


def _ctx():
    """The framework's context, made once by a program."""
    global _context
    import backup_1_b200 as b

    if _context is None:
        _context = b.Context(0)
    return _context


def _describe(code, scales, block_rows):
    import backup_1_b200 as b

    return b.Fp8Matrix.of(code, scales, block_rows)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    st = dict(case)
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        st["A"], st["sA"] = _quantised(_activations(g, m, k), case["a"], 1)
        st["B"], st["sB"] = _quantised(torch.randn(n, k, device=DEV, generator=g) * k ** -0.5, case["b"], case["b_rows"])
        st["C"] = torch.randn(m, n, device=DEV, generator=g).to(FLOAT[case["d"]]) if case["add"] else None
        st["D"] = torch.empty(m, n, device=DEV, dtype=FLOAT[case["d"]])
        if own:             # the descriptors that a program keeps beside its weights and buffers
            st["fA"], st["fB"] = _describe(st["A"], st["sA"], 1), _describe(st["B"], st["sB"], case["b_rows"])
        return st
    rows, cols, t = case["rows"], case["cols"], FLOAT[case["t"]]
    st["X"] = _activations(g, rows, cols).to(t)
    if case["op"] == "quant":
        st["Q"] = _empty_fp8(rows, cols, case["q"], case["block"])
        st["T"] = _empty_fp8(cols, rows, case["q"], case["block"]) if case["both"] else None
        if own:
            st["fQ"] = _describe(*st["Q"], case["block"])
            st["fT"] = _describe(*st["T"], case["block"]) if case["both"] else None
        return st
    st["R"] = torch.randn(rows, cols, device=DEV, generator=g).to(t) if case["res"] else None
    st["G"] = (1.0 + 0.1 * torch.randn(cols, device=DEV, generator=g)).to(t)
    if case["op"] == "norm":
        st["H"] = torch.empty(rows, cols, device=DEV, dtype=t) if case["res"] else None
        st["Y"] = torch.empty(rows, cols, device=DEV, dtype=t) if case["y"] else None
        st["Q"] = _empty_fp8(rows, cols, case["q"], 1)
        if own:
            st["fQ"] = _describe(*st["Q"], 1)
        return st
    st["dY"] = (0.1 * torch.randn(rows, cols, device=DEV, generator=g)).to(t)
    st["dX"] = torch.empty(rows, cols, device=DEV, dtype=t)
    st["dG"] = torch.empty(cols, device=DEV)
    if own:
        st["W"] = torch.empty(max(1, _ctx().rmsnorm_backward_workspace(rows, cols)), device=DEV, dtype=torch.uint8)
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------------
def _scales(amax, kind, rule):
    s = amax / FMAX[kind]
    if rule == "pow2":
        s = torch.exp2(torch.ceil(torch.log2(s)))
    return s.clamp_min(TINY)


def _quantise(x, kind, block_rows, rule):
    """Plain quantisation: the quotient in 64 bits, since values next to a rounding border turn over in 32."""
    rows, cols = x.shape
    s = _scales(_blocks(x, block_rows).abs().amax((1, 3)).double(), kind, rule).float()
    return (x.double() / _spread(s.double(), block_rows, rows, cols)).float().to(FP8[kind]), s


def run(st):
    if own:
        return _run_own(st)
    if st["op"] == "gemm":
        m, n, k = st["m"], st["n"], st["k"]
        a = st["A"].float() * _spread(st["sA"], 1, m, k)
        b = st["B"].float() * _spread(st["sB"], st["b_rows"], n, k)
        d = a @ b.t()
        if st["C"] is not None:
            d = d + st["C"].float()
        return {"D": d.to(FLOAT[st["d"]])}
    if st["op"] == "quant":
        x = st["X"].float()
        out = {}
        out["q"], out["s"] = _quantise(x, st["q"], st["block"], st["rule"])
        if st["both"]:
            out["qt"], out["st"] = _quantise(x.t(), st["q"], st["block"], st["rule"])
        return out
    t = FLOAT[st["t"]]
    if st["op"] == "norm":
        h = st["X"].float()
        out = {}
        if st["res"]:
            h = h + st["R"].float()
            out["h"] = h.to(t)
        y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * st["G"].float()
        if st["y"]:
            out["y"] = y.to(t)
        out["q"], out["s"] = _quantise(y, st["q"], 1, "amax")
        return out
    h, dy, gamma = st["X"].float(), st["dY"].float(), st["G"].float()
    r = torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)
    w = dy * gamma
    dx = r * (w - h * (r * r * (w * h).mean(1, keepdim=True)))
    if st["res"]:
        dx = dx + st["R"].float()
    return {"dx": dx.to(t), "dg": (dy * (h * r)).sum(0, dtype=torch.float64).float()}


def _run_own(st):
    import backup_1_b200 as b

    ctx, s = _ctx(), torch.cuda.current_stream()
    if st["op"] == "gemm":
        ctx.gemm_fp8(st["fA"], st["fB"], st["D"], st["n"], Cin=st["C"], ldc=st["n"], stream=s)
        return {"D": st["D"]}
    rows, cols = st["rows"], st["cols"]
    if st["op"] == "quant":
        rule = b.SCALE_POW2 if st["rule"] == "pow2" else b.SCALE_AMAX
        ctx.quantize_fp8(rows, cols, st["X"], cols, st["fQ"], st["fT"], rule=rule, stream=s)
        out = {"q": st["Q"][0], "s": st["Q"][1]}
        if st["both"]:
            out["qt"], out["st"] = st["T"]
        return out
    if st["op"] == "norm":
        ctx.rmsnorm(rows, cols, st["X"], cols, st["G"], EPS, R=st["R"], ldr=cols, H=st["H"], ldh=cols, Y=st["Y"], ldy=cols,
                    Q=st["fQ"], stream=s)
        out = {"q": st["Q"][0], "s": st["Q"][1]}
        if st["res"]:
            out["h"] = st["H"]
        if st["y"]:
            out["y"] = st["Y"]
        return out
    ctx.rmsnorm_backward(rows, cols, st["dY"], cols, st["X"], cols, st["G"], EPS, st["dX"], cols, st["dG"], dR=st["R"], lddr=cols,
                         workspace=st["W"], workspace_bytes=st["W"].numel(), stream=s)
    return {"dx": st["dX"], "dg": st["dG"]}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def _fp8_bytes(rows, cols, block_rows):
    return rows * cols + 4 * -(-rows // block_rows) * -(-cols // 128)


def work(case):
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        d = SIZE[case["d"]] * m * n
        return {"bytes": _fp8_bytes(m, k, 1) + _fp8_bytes(n, k, case["b_rows"]) + d * (2 if case["add"] else 1), "flops": 2.0 * m * n * k}
    rows, cols, e = case["rows"], case["cols"], SIZE[case["t"]]
    if case["op"] == "quant":
        b = e * rows * cols + _fp8_bytes(rows, cols, case["block"]) + (_fp8_bytes(cols, rows, case["block"]) if case["both"] else 0)
        return {"bytes": b, "flops": 4.0 * rows * cols}
    if case["op"] == "norm":
        arrays = 1 + 2 * case["res"] + case["y"]
        return {"bytes": e * rows * cols * arrays + e * cols + _fp8_bytes(rows, cols, 1), "flops": 8.0 * rows * cols}
    return {"bytes": e * rows * cols * (3 + case["res"]) + e * cols + 4 * cols, "flops": 12.0 * rows * cols}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------
def _codes64(v, kind):
    return v.float().to(FP8[kind]).double()


def _exact_fp8(x, kind, block_rows, rule):
    """Codes and scales block column by block column."""
    rows, cols = x.shape
    q = torch.empty(rows, cols, device=DEV, dtype=torch.float64)
    scales = []
    of_row = torch.arange(rows, device=DEV) // block_rows
    for c in range(0, cols, 128):
        part = x[:, c:c + 128]
        amax = torch.zeros(int(of_row[-1]) + 1, device=DEV, dtype=torch.float64).scatter_reduce(0, of_row, part.abs().amax(1), "amax")
        s = amax / FMAX[kind]
        if rule == "pow2":
            mant, e = torch.frexp(s)
            s = torch.ldexp(torch.ones_like(s), torch.where(mant > 0.5, e, e - 1))
        s = torch.maximum(s, torch.full_like(s, TINY))
        scales.append(s)
        q[:, c:c + 128] = _codes64(part / s.float().double()[of_row][:, None], kind)
    return q, torch.stack(scales, 1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        d = st["C"].double() if st["C"] is not None else torch.zeros(m, n, device=DEV, dtype=torch.float64)
        rows_b = torch.arange(n, device=DEV) // case["b_rows"]
        for kb in range(-(-k // 128)):
            part = st["A"][:, kb * 128:(kb + 1) * 128].double() @ st["B"][:, kb * 128:(kb + 1) * 128].double().t()
            part *= st["sA"][:, kb].double()[:, None]
            part *= st["sB"][:, kb].double()[rows_b][None, :]
            d += part
        return {"D": d}
    if case["op"] == "quant":
        out = {}
        out["q"], out["s"] = _exact_fp8(st["X"].double(), case["q"], case["block"], case["rule"])
        if case["both"]:
            out["qt"], out["st"] = _exact_fp8(st["X"].double().t(), case["q"], case["block"], case["rule"])
        return out
    if case["op"] == "norm":
        h = st["X"].double() + (st["R"].double() if case["res"] else 0.0)
        y = st["G"].double() * (h / torch.sqrt((h * h).sum(1, keepdim=True) / case["cols"] + EPS))
        out = {"h": h} if case["res"] else {}
        if case["y"]:
            out["y"] = y
        out["q"], out["s"] = _exact_fp8(y, case["q"], 1, "amax")
        return out
    h, dy, gamma = st["X"].double(), st["dY"].double(), st["G"].double()
    root = torch.sqrt((h * h).sum(1, keepdim=True) / case["cols"] + EPS)
    n = h / root                                     # the normalised row; dx is w's part that is not along it, over root
    w = dy * gamma
    dx = (w - n * ((w * n).sum(1, keepdim=True) / case["cols"])) / root
    if case["res"]:
        dx = dx + st["R"].double()
    return {"dx": dx, "dg": (dy * n).sum(0)}
