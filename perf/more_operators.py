"""Operators of a model's 8-bit block around the lm_head, measured on
device-resident buffers the way a serving loop calls them.

Four operators:
  norm     Sampler.block_norm_device: the end of one block and the start of the
           next, s = residual + scale * act(gate) * after(x), out = before(s)
  project  Sampler.matmul_int_device (and, for the lm_head, Sampler.gemv_device_ex
           with int8 weights): the product in 8-bit integers with a scale for
           each token and each output channel
  gated    Sampler.gated_int_device: both projections of a gated feed-forward,
           its activation and the product of the two
  ffn      a whole feed-forward block of them: the norm that quantises its
           tokens, the gated pair, the projection back, the norm behind it

Tokens are quantised symmetrically: scale = max|v| / 127 of the token,
q = v / scale rounded to the nearest integer, ties to even.

Every plain form is written in torch's elementary operations in binary32, but
for the quotient that an integer is rounded from, which is taken in binary64.
"""
import math

import torch

own = False

V = 151936                    # the workloads' vocabulary
MAX_NORM = 8192 * 4096        # what a drawn case may cost at most: elements,
MAX_WEIGHTS = V * 2048        # weights,
MAX_PRODUCT = 4096 * 4096 * 24576      # multiplications,
MAX_RESULTS = 4096 * 12288    # results
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
GGML = {"f32": 0, "f16": 1, "bf16": 30, "i8": 24}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
EPS = 1e-6


def listed():
    return [
        # a decode step of one sequence: residual sum and the next block's norm
        dict(name="norm-token", op="norm", m=1, c=4096, pad=0, x="bf16", res="bf16", out="bf16",
             after="none", before="rms", gate="none", act="none"),
        # a batch with norms on both sides and a gate of its own for every
        # token; an odd width, rows that start anywhere
        dict(name="norm-gated-300", op="norm", m=300, c=1001, pad=3, x="f16", res="f32", out="f16",
             after="layer", before="rms", gate="token", act="sigmoid"),
        # prompts, with a scale for each channel of the block's output: the largest norm
        dict(name="norm-prompts-8192", op="norm", m=8192, c=4096, pad=0, x="bf16", res="f32",
             out="bf16", after="rms", before="rms", gate="channel", act="none"),
        # the lm_head of one sequence, from float hidden states
        dict(name="lm-head-1", op="project", m=1, k=2048, n=V, pad=0, x="f32", out="f32",
             bias=False, head=True),
        # a decode batch through an inner projection, tokens quantised before
        dict(name="project-16", op="project", m=16, k=4096, n=4096, pad=0, x="i8", out="bf16",
             bias=False, head=False),
        # ragged sizes with a bias, float tokens quantised by the call
        dict(name="project-odd-77", op="project", m=77, k=1040, n=1001, pad=5, x="f16", out="f16",
             bias=True, head=False),
        # a few prompts through the projection back to the hidden width: long sums
        dict(name="project-prompts-4096", op="project", m=4096, k=12288, n=4096, pad=0, x="bf16",
             out="bf16", bias=False, head=False),
        # one token's gated pair
        dict(name="gated-1", op="gated", m=1, k=4096, n=12288, pad=0, x="bf16", out="f32",
             act="silu"),
        # a small batch, odd sizes
        dict(name="gated-odd-33", op="gated", m=33, k=1040, n=2731, pad=16, x="i8", out="f16",
             act="gelu"),
        # prompts: the largest product
        dict(name="gated-prompts-4096", op="gated", m=4096, k=4096, n=12288, pad=0, x="i8",
             out="bf16", act="silu"),
        # a whole feed-forward block of a decode batch
        dict(name="ffn-8", op="ffn", m=8, c=2048, n=8192, act="silu"),
        # and of a prompt
        dict(name="ffn-prompt-1500", op="ffn", m=1500, c=4096, n=8192, act="gelu_tanh"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["norm", "project", "project", "gated", "ffn"])
    f = ["f32", "f16", "bf16"]
    if op == "norm":
        c = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            c = max(8, c // 8 * 8)
        m = _log(rng, 1, min(8192, MAX_NORM // c))
        gate = rng.choice(["none", "channel", "token"])
        return dict(op=op, m=m, c=c, pad=rng.choice([0, 0, 8, 3]), x=rng.choice(f), res=rng.choice(f),
                    out=rng.choice(f), after=rng.choice(["none", "rms", "layer"]),
                    before=rng.choice(["rms", "layer"]), gate=gate,
                    act=rng.choice(["none", "sigmoid", "tanh"]) if gate != "none" else "none")
    k = 16 * _log(rng, 4, 768)
    if op == "ffn":
        m, c = _log(rng, 1, 2048), 16 * _log(rng, 8, 256)
        return dict(op=op, m=m, c=c, n=16 * _log(rng, 16, 768), act=rng.choice(["silu", "gelu", "gelu_tanh"]))
    pair = 2 if op == "gated" else 1
    n = _log(rng, 64, min(V, MAX_WEIGHTS // (pair * k)))
    m = _log(rng, 1, max(1, min(4096, MAX_RESULTS // n, MAX_PRODUCT // (pair * k * n))))
    x = rng.choice(["i8", "i8", "f32", "f16", "bf16"])
    pad = rng.choice([0, 0, 16, 32]) if x == "i8" else rng.choice([0, 0, 8, 5])
    c = dict(op=op, m=m, k=k, n=n, pad=pad, x=x, out=rng.choice(f))
    if op == "gated":
        c["act"] = rng.choice(["silu", "gelu", "gelu_tanh", "relu"])
    else:
        c["head"] = x == "f32" and c["out"] == "f32" and rng.random() < 0.5
        c["bias"] = not c["head"] and rng.random() < 0.4
    return c


# ---- inputs ---------------------------------------------------------------

def _rows(m, c, pad, kind, g, big=0.004, std=1.0):
    """Tokens as a model has them, some channels far above the others, in rows
    a little longer than they are wide."""
    far = torch.rand(c, device="cuda", generator=g) < big
    x = torch.empty(m, c, device="cuda").normal_(0.0, std, generator=g)
    x = torch.where(far, x * 12.0, x).to(DTYPES[kind])
    return _padded(x, pad)


def _padded(x, pad):
    if not pad:
        return x.contiguous()
    whole = torch.zeros(x.shape[0], x.shape[1] + pad, device="cuda", dtype=x.dtype)
    whole[:, : x.shape[1]] = x
    return whole


def _int8_rows(v):
    scale = v.abs().amax(-1) / 127.0
    return (v / scale[:, None]).round().to(torch.int8), scale


def _weights(n, k, g):
    """int8 rows of an output channel each, and their scales."""
    w = torch.empty(n, k, device="cuda", dtype=torch.int8)
    s = torch.empty(n, device="cuda")
    for at in range(0, n, 16384):
        part = torch.empty(min(16384, n - at), k, device="cuda").normal_(0.0, k ** -0.5, generator=g)
        w[at:at + 16384], s[at:at + 16384] = _int8_rows(part)
    return w, s


def _near_one(c, g):
    return torch.empty(c, device="cuda").normal_(1.0, 0.2, generator=g)


def _norm_of(kind, c, g):
    s = {}
    if kind != "none":
        s["w"] = _near_one(c, g)
    if kind == "layer":
        s["b"] = torch.empty(c, device="cuda").normal_(0.0, 0.2, generator=g)
    return s


def _inputs(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed * 7919 + case["m"])
    op, m = case["op"], case["m"]
    if op == "norm":
        c, pad = case["c"], case["pad"]
        s = dict(x=_rows(m, c, pad, case["x"], g), res=_rows(m, c, pad, case["res"], g, std=3.0),
                 after=_norm_of(case["after"], c, g), before=_norm_of(case["before"], c, g))
        if case["gate"] != "none":
            s["gate"] = _rows(m if case["gate"] == "token" else 1, c, pad, case["x"], g, 0.0)
        return s
    if op == "ffn":
        c, n = case["c"], case["n"]
        return dict(x=_rows(m, c, 0, "bf16", g), res=_rows(m, c, 0, "bf16", g, std=3.0),
                    before=_near_one(c, g), after=_near_one(c, g), next=_near_one(c, g),
                    w=_weights(n, c, g), up=_weights(n, c, g), down=_weights(c, n, g))
    k, n = case["k"], case["n"]
    if case["x"] == "i8":
        q, scale = _int8_rows(_rows(m, k, 0, "f32", g))
        s = dict(x=_padded(q, case["pad"]), xs=scale)
    else:
        s = dict(x=_rows(m, k, case["pad"], case["x"], g))
    s["w"] = _weights(n, k, g)
    if op == "gated":
        s["up"] = _weights(n, k, g)
    elif case["bias"]:
        s["bias"] = torch.empty(n, device="cuda").normal_(0.0, 0.5, generator=g)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    m, dev = case["m"], "cuda"
    if case["op"] == "norm":
        c = case["c"] + case["pad"]
        s["sum"] = torch.zeros(m, c, device=dev, dtype=DTYPES[case["res"]])
        s["out"] = torch.zeros(m, c, device=dev, dtype=DTYPES[case["out"]])
    elif case["op"] == "ffn":
        c, n = case["c"], case["n"]
        s["mid"] = torch.empty(m, c, device=dev)
        s["q"] = torch.empty(m, c, device=dev, dtype=torch.int8)
        s["qs"] = torch.empty(m, device=dev)
        s["h"] = torch.empty(m, n, device=dev, dtype=torch.int8)
        s["hs"] = torch.empty(m, device=dev)
        s["y"] = torch.empty(m, c, device=dev)
        s["sum"] = torch.empty(m, c, device=dev, dtype=torch.bfloat16)
        s["out"] = torch.empty(m, c, device=dev, dtype=torch.bfloat16)
    else:
        s["y"] = torch.empty(m, case["n"], device=dev, dtype=DTYPES[case["out"]])
    return s


# ---- the plain forms --------------------------------------------------------

def _act(v, kind):
    if kind == "silu":
        return v / (1.0 + torch.exp(-v))
    if kind == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if kind == "relu":
        return torch.where(v > 0, v, 0.0)
    if kind == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-v))
    return torch.tanh(v) if kind == "tanh" else v


def _norm(v, kind, p):
    if kind == "none":
        return v
    if kind == "rms":
        return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * p["w"]
    v = v - v.mean(-1, keepdim=True)
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * p["w"] + p["b"]


def _quantised(v):
    scale = v.abs().amax(-1, keepdim=True) / 127.0
    return (v.double() / scale.double()).round().float(), scale


def _product(q, scale, w):
    return q @ w[0].float().t() * scale * w[1]


def _plain_norm(s):
    c = s["case"]
    n = c["c"]
    y = _norm(s["x"][:, :n].float(), c["after"], s["after"])
    if c["gate"] != "none":
        y = y * _act(s["gate"][:, :n].float(), c["act"])
    t = s["res"][:, :n].float() + 0.7 * y
    out = _norm(t, c["before"], s["before"])
    return dict(sum=t.to(DTYPES[c["res"]]), out=out.to(DTYPES[c["out"]]))


def _tokens(s):
    c = s["case"]
    x = s["x"][:, : c["k"]].float()
    return (x, s["xs"][:, None]) if c["x"] == "i8" else _quantised(x)


def _plain_project(s):
    q, scale = _tokens(s)
    y = _product(q, scale, s["w"])
    if s["case"]["bias"]:
        y = y + s["bias"]
    return y.to(DTYPES[s["case"]["out"]])


def _plain_gated(s):
    q, scale = _tokens(s)
    y = _act(_product(q, scale, s["w"]), s["case"]["act"]) * _product(q, scale, s["up"])
    return y.to(DTYPES[s["case"]["out"]])


def _plain_ffn(s):
    mid = s["res"].float() + s["x"].float()
    q, scale = _quantised(_norm(mid, "rms", dict(w=s["before"])))
    h = _act(_product(q, scale, s["w"]), s["case"]["act"]) * _product(q, scale, s["up"])
    y = _product(*_quantised(h), s["down"])
    t = mid + 0.7 * _norm(y, "rms", dict(w=s["after"]))
    out = _norm(t, "rms", dict(w=s["next"]))
    return dict(mid=mid, sum=t.bfloat16(), out=out.bfloat16())


# ---- the framework's operators --------------------------------------------------

_SAMPLER = None


def _calls(s):
    """The descriptors over the state's buffers, made once as a serving loop
    makes them for the buffers that it keeps."""
    global _SAMPLER
    from hachiue_amd import Sampler
    from hachiue_amd import sampler as hs
    if _SAMPLER is None:
        _SAMPLER = Sampler(0)
    S, c, st = _SAMPLER, s["case"], torch.cuda.current_stream().cuda_stream
    kinds = {"none": hs.NORM_NONE, "rms": hs.NORM_RMS, "layer": hs.NORM_LAYER}
    acts = {"none": hs.ACT_NONE, "silu": hs.ACT_SILU, "gelu": hs.ACT_GELU,
            "gelu_tanh": hs.ACT_GELU_TANH, "relu": hs.ACT_RELU, "sigmoid": hs.ACT_SIGMOID,
            "tanh": hs.ACT_TANH}
    names = {v: k for k, v in DTYPES.items()}

    def rows(t, scales=None):
        return hs.rows(GGML[names[t.dtype]], t.data_ptr(), t.shape[1],
                       None if scales is None else scales.data_ptr())

    def weights(w):
        return hs.weights(GGML["i8"], w[0].shape[0], w[0].shape[1], w[0].data_ptr(), w[1].data_ptr())

    def norm(kind, w=None, b=None):
        return hs.norm(kinds[kind], EPS, None if w is None else w.data_ptr(),
                       None if b is None else b.data_ptr())

    m = c["m"]
    if c["op"] == "norm":
        gate = None
        if c["gate"] != "none":
            gate = rows(s["gate"])
            if c["gate"] == "channel":
                gate.stride = 0
        block = hs.block_norm(m, c["c"], rows(s["x"]), residual=rows(s["res"]), scale=0.7,
                              gate=gate, gate_act=acts[c["act"]], sum=rows(s["sum"]),
                              after=norm(c["after"], **s["after"]),
                              before=norm(c["before"], **s["before"]), out=rows(s["out"]))
        return [(S.block_norm_device, (block, st))]
    if c["op"] == "ffn":
        w, up, down = weights(s["w"]), weights(s["up"]), weights(s["down"])
        q, h, y, mid = rows(s["q"], s["qs"]), rows(s["h"], s["hs"]), rows(s["y"]), rows(s["mid"])
        first = hs.block_norm(m, c["c"], rows(s["x"]), residual=rows(s["res"]), sum=mid,
                              before=norm("rms", s["before"]), out=q)
        last = hs.block_norm(m, c["c"], y, residual=mid, scale=0.7, sum=rows(s["sum"]),
                             after=norm("rms", s["after"]), before=norm("rms", s["next"]),
                             out=rows(s["out"]))
        return [(S.block_norm_device, (first, st)),
                (S.gated_int_device, (m, q, w, up, acts[c["act"]], h, st)),
                (S.matmul_int_device, (m, h, down, None, y, st)),
                (S.block_norm_device, (last, st))]
    x, y = rows(s["x"], s.get("xs")), rows(s["y"])
    if c["op"] == "gated":
        return [(S.gated_int_device, (m, x, weights(s["w"]), weights(s["up"]), acts[c["act"]], y, st))]
    if c["head"]:
        return [(S.gemv_device_ex, (s["x"].data_ptr(), m, s["x"].shape[1], weights(s["w"]),
                                    s["y"].data_ptr(), c["n"], st))]
    bias = s["bias"].data_ptr() if c["bias"] else None
    return [(S.matmul_int_device, (m, x, weights(s["w"]), bias, y, st))]


def run(s):
    c = s["case"]
    if not own:
        return dict(norm=_plain_norm, project=_plain_project, gated=_plain_gated,
                    ffn=_plain_ffn)[c["op"]](s)
    if "calls" not in s:
        s["calls"] = _calls(s)
    for f, args in s["calls"]:
        f(*args)
    if c["op"] == "norm":
        return dict(sum=s["sum"][:, : c["c"]], out=s["out"][:, : c["c"]])
    if c["op"] == "ffn":
        return dict(mid=s["mid"], sum=s["sum"], out=s["out"])
    return s["y"]


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    """norm: every tensor once.  project, gated: tokens, weights and scales
    read once, results written once.  ffn: the block's input and output rows
    and its weights; what the block keeps to itself is not counted."""
    m = case["m"]
    if case["op"] == "norm":
        c = case["c"]
        gates = {"none": 0, "channel": 1, "token": m}[case["gate"]] * c * SIZE[case["x"]]
        par = 4 * c * sum({"none": 0, "rms": 1, "layer": 2}[case[p]] for p in ("after", "before"))
        each = SIZE[case["x"]] + 2 * SIZE[case["res"]] + SIZE[case["out"]]
        return dict(bytes=m * c * each + gates + par, flops=12 * m * c)
    n = case["n"]
    if case["op"] == "ffn":
        c = case["c"]
        return dict(bytes=m * c * (2 + 2 + 4 + 2 + 2) + 3 * n * c + 4 * (2 * n + c) + 12 * c,
                    flops=6 * m * n * c)
    k, pair = case["k"], 2 if case["op"] == "gated" else 1
    tokens = m * k * SIZE[case["x"]] + (4 * m if case["x"] == "i8" else 0)
    return dict(bytes=tokens + pair * (n * k + 4 * n) + (4 * n if case.get("bias") else 0) +
                m * n * SIZE[case["out"]], flops=2 * pair * m * n * k)


# ---- the same in 64 bits ------------------------------------------------------

_ACT64 = {
    "none": lambda v: v,
    "silu": lambda v: v * torch.sigmoid(v),
    "gelu": lambda v: v * 0.5 * torch.special.erfc(-v / 2 ** 0.5),
    "gelu_tanh": lambda v: v * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (v + 0.044715 * v ** 3)),
    "relu": lambda v: v.clamp(min=0.0),
    "sigmoid": torch.sigmoid,
    "tanh": torch.tanh,
}


def _norm64(v, kind, p):
    if kind == "none":
        return v
    mean = v.sum(1) / v.shape[1] if kind == "layer" else torch.zeros(v.shape[0], device=v.device).double()
    d = v - mean[:, None]
    d = d / torch.sqrt((d ** 2).sum(1) / v.shape[1] + EPS)[:, None] * p["w"].double()
    return d + p["b"].double() if kind == "layer" else d


def _round64(v):
    """A token's integers and its scale, the largest magnitude over 127 as it
    is held in 32 bits."""
    scale = (v.abs().max(1).values.float() / 127.0).double()
    return torch.round(v / scale[:, None]), scale


def _dot64(q, scale, w):
    y = torch.empty(q.shape[0], w[0].shape[0], dtype=torch.float64, device=q.device)
    for at in range(0, w[0].shape[0], 16384):
        part = w[0][at:at + 16384].double()
        y[:, at:at + 16384] = q @ part.t()
    return y * scale[:, None] * w[1].double()[None]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "norm":
        c = case["c"]
        y = _norm64(s["x"][:, :c].double(), case["after"], s["after"])
        if case["gate"] != "none":
            y = _ACT64[case["act"]](s["gate"][:, :c].double()) * y
        t = y * 0.7 + s["res"][:, :c].double()
        return dict(sum=t, out=_norm64(t, case["before"], s["before"]))
    act = _ACT64.get(case.get("act", "none"))
    if case["op"] == "ffn":
        mid = s["x"].double() + s["res"].double()
        q, scale = _round64(_norm64(mid, "rms", dict(w=s["before"])))
        h = act(_dot64(q, scale, s["w"])) * _dot64(q, scale, s["up"])
        y = _norm64(_dot64(*_round64(h), s["down"]), "rms", dict(w=s["after"]))
        t = y * 0.7 + mid
        return dict(mid=mid, sum=t, out=_norm64(t, "rms", dict(w=s["next"])))
    x = s["x"][:, : case["k"]].double()
    q, scale = (x, s["xs"].double()) if case["x"] == "i8" else _round64(x)
    y = _dot64(q, scale, s["w"])
    if case["op"] == "gated":
        return act(y) * _dot64(q, scale, s["up"])
    return y + s["bias"].double() if case["bias"] else y
