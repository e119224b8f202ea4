"""What the sequence operators of the recogniser are measured on: a matrix product with its epilogue (`linear`), attention
over the states of lines of different lengths (`cross_attention`) and the norm with the residual's addition (`rms_norm`).

`run` computes them in elementary torch operations, or with `own` set through `ocr_amd.crnn.network_hip.CRNN`."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
E4M3_MAX = 448.0
T_LINE = 71            # timesteps of a line of width 280
EPS = 1e-6


def listed():
    return [
        # one row of a decoder's step through a 512-wide projection with the residual: launch latency
        dict(name="linear 1 row", op="linear", m=1, k=512, n=512, dtype="bf16", act="none", bias=True, residual=True),
        # the crops of one page, one step each, through the 5530-class output layer (an odd number of columns)
        dict(name="linear 48 rows 5530 classes", op="linear", m=48, k=512, n=5530, dtype="bf16", act="none", bias=True, residual=False),
        # every state of 256 lines of width 280 into a 2048-wide hidden layer
        dict(name="linear states up", op="linear", m=256 * T_LINE, k=512, n=2048, dtype="bf16", act="gelu", bias=True, residual=False),
        # a wide layer over many rows: the matrix cores' own rate
        dict(name="linear wide", op="linear", m=16384, k=4096, n=4096, dtype="bf16", act="none", bias=True, residual=True),
        # 64 lines' states in the recogniser's default precision
        dict(name="linear fp32", op="linear", m=64 * T_LINE, k=512, n=512, dtype="fp32", act="relu", bias=True, residual=True),
        # 8-bit operands as the norm leaves them, 256 lines' states through a 2048-wide layer
        dict(name="linear 8 bits", op="linear", m=256 * T_LINE, k=2048, n=2048, dtype="e4m3", act="silu", bias=True, residual=True),
        # a decoder's step for 8 lines: latency
        dict(name="norm 8 rows", op="norm", m=8, n=512, dtype="bf16", out="bf16", residual=True),
        # the rows that feed the 8-bit product
        dict(name="norm to 8 bits", op="norm", m=256 * T_LINE, n=2048, dtype="bf16", out="e4m3", residual=True),
        # one decoding step for 256 lines: each query row reads its own line's states
        dict(name="attention step", op="attention", b=256, tq=1, tk=T_LINE, hkv=8, group=1, d=64, dtype="bf16", lengths=True, mask=False),
        # a query over all states of a batch of lines laid end to end, the padding steps of each line masked out
        dict(name="attention long memory", op="attention", b=2, tq=1, tk=256 * T_LINE, hkv=8, group=1, d=64, dtype="bf16", lengths=False, mask=True),
        # many queries, long states, four query heads to a key head: the matrix cores' rate
        dict(name="attention many rows", op="attention", b=8, tq=1024, tk=4096, hkv=4, group=4, d=128, dtype="bf16", lengths=True, mask=False),
        # a decoder's whole text (48 characters) over its line, in the recogniser's default precision
        dict(name="attention fp32", op="attention", b=64, tq=48, tk=T_LINE, hkv=8, group=1, d=64, dtype="fp32", lengths=True, mask=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "attention", "attention"])
    if op == "linear":
        dtype = rng.choice(["bf16", "bf16", "e4m3", "fp32"])
        k, n = _log(rng, 64, 8192), _log(rng, 32, 8192)
        if rng.random() < 0.75:              # most layers have round widths
            k, n = -(-k // 64) * 64, -(-n // 16) * 16
        most = 2.5e10 if dtype == "fp32" else 2.5e11
        m = _log(rng, 1, max(1, min(20000, int(most / k / n))))
        return dict(op=op, m=m, k=k, n=n, dtype=dtype, act=rng.choice(["none", "relu", "leaky", "gelu", "silu"]),
                    bias=rng.random() < 0.7, residual=rng.random() < 0.5)
    if op == "norm":
        n = _log(rng, 64, 8192)
        if rng.random() < 0.75:
            n = -(-n // 64) * 64
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        return dict(op=op, m=_log(rng, 1, max(1, int(3.5e7 / n))), n=n, dtype=dtype, out=rng.choice([dtype, "e4m3"]), residual=rng.random() < 0.7)
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    d, hkv, group = rng.choice([32, 64, 64, 128, 80]), rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4])
    tk = _log(rng, 1, 18176)
    b = _log(rng, 1, max(1, min(256, int(1e8 / (tk * hkv * d)))))
    most = min(1e8 if dtype == "fp32" else 5e8, (1.5e10 if dtype == "fp32" else 1.3e11) / d) / (b * hkv * group * tk)
    tq = _log(rng, 1, max(1, min(1024, int(most))))
    return dict(op=op, b=b, tq=tq, tk=tk, hkv=hkv, group=group, d=d, dtype=dtype, lengths=rng.random() < 0.7, mask=rng.random() < 0.3)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dev = "cuda"

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    c = dict(case)
    if c["op"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        x, w = torch.tanh(normal(m, k)), normal(n, k) / math.sqrt(k)       # states lie in [-1, 1]
        s = dict(case=c, x_scale=None, w_scale=None)
        if c["dtype"] == "e4m3":                                           # a scale a row of x and a column of the result
            for name, t in (("x", x), ("w", w)):
                top = t.abs().amax(1).clamp_min(1e-30) / E4M3_MAX
                s[name], s[name + "_scale"] = (t / top[:, None]).to(torch.float8_e4m3fn), top
        else:
            s["x"], s["w"] = x.to(DTYPES[c["dtype"]]), w.to(DTYPES[c["dtype"]])
        s["out"] = torch.float32 if c["dtype"] == "fp32" else torch.bfloat16
        s["bias"] = 0.5 * normal(n) if c["bias"] else None
        s["residual"] = normal(m, n).to(s["out"]) if c["residual"] else None
        return s
    if c["op"] == "norm":
        m, n, dt = c["m"], c["n"], DTYPES[c["dtype"]]
        x = (normal(m, n) * torch.exp(0.5 * normal(m, 1))).to(dt)
        return dict(case=c, x=x, residual=(0.5 * normal(m, n)).to(dt) if c["residual"] else None, gain=1 + 0.2 * normal(n), out=DTYPES[c["out"]])
    b, tq, tk, hkv, hq, d, dt = c["b"], c["tq"], c["tk"], c["hkv"], c["hkv"] * c["group"], c["d"], DTYPES[c["dtype"]]
    q = (1.5 * normal(b, tq, hq, d)).to(dt)
    kv = normal(b, tk, 2, hkv, d).to(dt)                                   # one projection gives both: keys and values interleaved
    lengths = mask = None
    if c["lengths"]:
        lengths = torch.randint(min(tk, max(1, tk // 3)), tk + 1, (b,), generator=g, device=dev, dtype=torch.int32)
    if c["mask"]:                                                          # lines of T_LINE steps end to end, each with its own valid part
        lines = -(-tk // T_LINE)
        valid = torch.randint(2, T_LINE + 1, (b, lines, 1), generator=g, device=dev)
        mask = (torch.arange(T_LINE, device=dev)[None, None] < valid).reshape(b, -1)[:, :tk].contiguous()
    return dict(case=c, q=q, k=kv[:, :, 0], v=kv[:, :, 1], lengths=lengths, mask=mask)


_reader = []


def _crnn():
    """The recogniser's handle, as a program that uses it holds one."""
    if not _reader:
        from ocr_amd.crnn.network_hip import CRNN
        _reader.append(CRNN(32, 1, 65, 256, device=torch.cuda.current_device()))
    return _reader[0]


def _linear(s):
    y = s["x"].float() @ s["w"].float().t()
    if s["x_scale"] is not None:
        y = y * s["x_scale"][:, None] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    act = s["case"]["act"]
    if act == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif act == "leaky":
        y = torch.where(y > 0, y, 0.2 * y)
    elif act == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    elif act == "silu":
        y = y / (1 + torch.exp(-y))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["out"])


def _norm(s):
    t = s["x"].float()
    if s["residual"] is not None:
        t = t + s["residual"].float()
    y = t * torch.rsqrt((t * t).mean(1, keepdim=True) + EPS) * s["gain"]
    got = {"sum": t.to(s["x"].dtype)} if s["residual"] is not None else {}
    if s["out"] is torch.float8_e4m3fn:
        scale = y.abs().amax(1).clamp_min(E4M3_MAX * 2.0 ** -126) / E4M3_MAX
        got["y"], got["scale"] = (y / scale[:, None]).to(s["out"]), scale
    else:
        got["y"] = y.to(s["out"])
    return got


def _attention(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    b, tq, hq, d = q.shape
    tk, hkv = k.shape[1], k.shape[2]
    q = q.view(b, tq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b * hkv, -1, d)
    k, v = (t.permute(0, 2, 1, 3).reshape(b * hkv, tk, d) for t in (k, v))
    p = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(d ** -0.5).view(b, hkv, -1, tk)
    ok = torch.ones(b, tk, dtype=torch.bool, device=q.device)
    if s["lengths"] is not None:
        ok = ok & (torch.arange(tk, device=q.device) < s["lengths"][:, None])
    if s["mask"] is not None:
        ok = ok & s["mask"]
    p.masked_fill_(~ok[:, None, None], -math.inf)
    top = p.amax(3, keepdim=True).clamp_min(-3e38)
    p = p.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    o = torch.matmul(p.view(b * hkv, -1, tk), v).view(b, hkv, -1, d) / torch.where(total > 0, total, torch.ones_like(total))
    return o.view(b, hkv, hq // hkv, tq, d).permute(0, 3, 1, 2, 4).reshape(b, tq, hq, d).to(s["q"].dtype)


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"linear": _linear, "norm": _norm, "attention": _attention}[op](s)
    c = _crnn()
    if op == "linear":
        return c.linear(s["x"], s["w"], bias=s["bias"], residual=s["residual"], act=s["case"]["act"], x_scale=s["x_scale"], w_scale=s["w_scale"])
    if op == "norm":
        got = c.rms_norm(s["x"], s["gain"], residual=s["residual"], eps=EPS, out_dtype=s["out"])
        return {k: v for k, v in got._asdict().items() if v is not None}
    return c.cross_attention(s["q"], s["k"], s["v"], lengths=s["lengths"], mask=s["mask"])


def work(case):
    c, size = case, {"fp32": 4, "bf16": 2, "e4m3": 1}
    e = size[c["dtype"]]
    if c["op"] == "linear":
        m, n, k, eo = c["m"], c["n"], c["k"], 4 if c["dtype"] == "fp32" else 2
        extra = (4 * (m + n) if c["dtype"] == "e4m3" else 0) + (4 * n if c["bias"] else 0) + (m * n * eo if c["residual"] else 0)
        return {"bytes": (m + n) * k * e + m * n * eo + extra, "flops": 2 * m * n * k}
    if c["op"] == "norm":
        m, n = c["m"], c["n"]
        return {"bytes": m * n * (e * (3 if c["residual"] else 1) + size[c["out"]]) + 4 * n + (4 * m if c["out"] == "e4m3" else 0), "flops": 6 * m * n}
    keys = c["b"] * c["tk"] * (2 / 3 if c["lengths"] else 1) * (0.51 if c["mask"] else 1)       # the mean part that is read
    hq = c["hkv"] * c["group"]
    return {"bytes": e * c["d"] * (2 * keys * c["hkv"] + 2 * c["b"] * c["tq"] * hq) + (c["b"] * c["tk"] if c["mask"] else 0),
            "flops": 4 * keys * c["tq"] * hq * c["d"]}


def exact(case, seed):
    """The definitions in 64 bits, head by head and row block by row block."""
    s = prepare(case, seed)
    if case["op"] == "linear":
        w = s["w"].double() if s["w_scale"] is None else s["w"].double() * s["w_scale"].double()[:, None]
        wt, rows = w.t().contiguous(), []
        for at in range(0, case["m"], 4096):
            x = s["x"][at:at + 4096].double()
            z = x @ wt if s["x_scale"] is None else (x * s["x_scale"][at:at + 4096].double()[:, None]) @ wt
            if s["bias"] is not None:
                z += s["bias"].double()
            z = {"none": lambda t: t, "relu": lambda t: t.clamp(min=0), "leaky": lambda t: torch.maximum(t, 0.2 * t),
                 "gelu": lambda t: t * 0.5 * torch.erfc(-t / math.sqrt(2.0)), "silu": lambda t: t * torch.sigmoid(t)}[case["act"]](z)
            rows.append(z if s["residual"] is None else z + s["residual"][at:at + 4096].double())
        return torch.cat(rows)
    if case["op"] == "norm":
        t = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        y = t / (t.square().sum(1, keepdim=True) / case["n"] + EPS).sqrt() * s["gain"].double()
        got = {} if s["residual"] is None else {"sum": t}
        if case["out"] != "e4m3":
            return dict(got, y=y)
        c = (y.abs().max(1).values / E4M3_MAX).clamp(min=2.0 ** -126)
        z = y / c[:, None]                                  # to the nearest of 8 steps a power of two, subnormal ones below 2^-6
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
        return dict(got, y=torch.round(z / step) * step, scale=c)
    q, k, v = s["q"], s["k"], s["v"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group = case["group"]
    for i in range(case["b"]):
        n = case["tk"] if s["lengths"] is None else int(s["lengths"][i])
        at = torch.arange(n, device=q.device)
        if s["mask"] is not None:
            at = at[s["mask"][i, :n]]
        if at.numel() == 0:
            continue
        ki, vi, qi = k[i, at].double(), v[i, at].double(), q[i].double()
        for h in range(case["hkv"]):
            rows = qi[:, h * group:(h + 1) * group].reshape(-1, case["d"])
            p = torch.softmax(rows @ ki[:, h].t().contiguous() / math.sqrt(case["d"]), dim=1)
            out[i, :, h * group:(h + 1) * group] = (p @ vi[:, h].contiguous()).view(case["tq"], group, case["d"])
    return out
