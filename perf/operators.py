"""The 8-bit integer LM head and the beam-search step, as cases to measure.

Five operators of one decode step of beam search, in the order in which a program runs them:

  quantize  capi.quantize_rows_i8  rows to int8 codes with one scale for each row, optionally
                                   RMS-normalised first (weights once, activations each step)
  matmul    capi.matmul_i8         out[m][n] = a_scale[m] b_scale[n] sum_k a[m][k] b[n][k]
  lmhead    capi.lmhead_logits_i8  final norm, quantisation, int8 product, softcap: the logits
  select    capi.beam_select       the k best continuations over beams and vocabulary
  reorder   capi.beam_reorder      states (caches, histories) moved after the chosen parents

`run` computes them in elementary torch operations while `own` is false, and calls the library
while it is true.  `exact` states each once more in 64 bits.
"""
import math

import torch

own = False

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = {"f32": F32, "bf16": BF16, "f16": F16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4}
EPS = 1e-6


def listed():
    return [
        # one decode step's hidden states before a projection: latency
        dict(name="quantize 4x4096 f32 norm", op="quantize", rows=4, cols=4096, dtype="f32", norm=True),
        # an output matrix taken to int8 when a model is loaded: bandwidth
        dict(name="quantize 32000x4096 bf16", op="quantize", rows=32000, cols=4096, dtype="bf16", norm=False),
        # a projection for a small batch of sequences
        dict(name="matmul 16x4096x4096 bf16", op="matmul", m=16, n=4096, k=4096, out="bf16"),
        # a projection over a prompt's tokens: bound by the matrix unit
        dict(name="matmul 2048x8192x8192 bf16", op="matmul", m=2048, n=8192, k=8192, out="bf16"),
        # one sequence's logits: the weights are read once
        dict(name="lmhead 1x4096x128256", op="lmhead", rows=1, hidden=4096, vocab=128256, add_one=False, softcap=0.0),
        # 32 sequences of 8 beams, (w + 1) norm and softcap, the widest vocabulary
        dict(name="lmhead 256x2304x256000 cap", op="lmhead", rows=256, hidden=2304, vocab=256000, add_one=True,
             softcap=30.0),
        # one sequence of 4 beams on a small vocabulary: latency
        dict(name="select 1x4x32000 f32", op="select", batch=1, beams=4, vocab=32000, k=8, dtype="f32", allowed=1.0,
             finished=0.0, alpha=0.0, first=False),
        # a few sequences, twice as many continuations as beams, bf16 logits of an odd width
        dict(name="select 8x4x128257 bf16", op="select", batch=8, beams=4, vocab=128257, k=8, dtype="bf16",
             allowed=1.0, finished=0.0, alpha=0.0, first=False),
        # constrained decoding: 2 % of the ids allowed, some beams ended, length-normalised ranks
        dict(name="select 16x8x151936 masked", op="select", batch=16, beams=8, vocab=151936, k=8, dtype="f32",
             allowed=0.02, finished=0.25, alpha=0.6, first=False),
        # 512 rows of the widest vocabulary: bandwidth
        dict(name="select 64x8x262144 bf16", op="select", batch=64, beams=8, vocab=262144, k=16, dtype="bf16",
             allowed=1.0, finished=0.0, alpha=0.0, first=False),
        # the token histories of one sequence's beams, an odd length: latency
        dict(name="reorder ids 1x4x511", op="reorder", batch=1, beams=4, tensors=1, heads=1, cap=511, length=511, dim=1,
             dtype="i32", moved=2),
        # keys and values of eight layers, the used part of a cache: bandwidth
        dict(name="reorder kv 8x8 8 layers", op="reorder", batch=8, beams=8, tensors=16, heads=8, cap=1024, length=1000,
             dim=128, dtype="bf16", moved=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 200)


def draw(rng):
    op = rng.choice(["quantize", "matmul", "lmhead", "select", "select", "reorder"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        if op == "quantize":
            c = dict(op=op, rows=_log(rng, 1, 32768), cols=_log(rng, 200, 8192), dtype=rng.choice(["f32", "bf16", "f16"]),
                     norm=rng.random() < 0.5)
        elif op == "matmul":
            c = dict(op=op, m=_log(rng, 1, 2048), n=_log(rng, 500, 16384), k=_log(rng, 200, 8192),
                     out=rng.choice(["f32", "bf16", "f16"]))
        elif op == "lmhead":
            c = dict(op=op, rows=_log(rng, 1, 256), hidden=_log(rng, 1000, 8192), vocab=_log(rng, 16000, 262144),
                     add_one=rng.random() < 0.3, softcap=rng.choice([0.0, 30.0]))
        elif op == "select":
            beams = rng.randint(1, 16)
            c = dict(op=op, batch=_log(rng, 1, 64), beams=beams, vocab=_log(rng, 16000, 262144),
                     k=beams * rng.choice([1, 2]), dtype=rng.choice(["f32", "bf16", "f16"]),
                     allowed=rng.choice([1.0, 1.0, 0.1, 0.02]), finished=rng.choice([0.0, 0.0, 0.25]),
                     alpha=rng.choice([0.0, 0.6, 1.0]), first=rng.random() < 0.1)
        else:
            beams = rng.randint(2, 16)
            cap = _log(rng, 64, 4096)
            c = dict(op=op, batch=_log(rng, 1, 32), beams=beams, tensors=rng.choice([1, 2, 8, 16]), heads=_log(rng, 1, 16),
                     cap=cap, length=rng.randint(cap // 2, cap), dim=rng.choice([1, 64, 80, 128]),
                     dtype=rng.choice(["f32", "bf16"]), moved=rng.randint(1, beams))
        if _cost(c) <= most:
            return c


def _sources(c):
    """How many different beams the moved ones of one sequence are expected to come from."""
    b = c["beams"]
    return b * (1 - (1 - 1 / b) ** c["moved"])


def work(case):
    c, op = case, case["op"]
    if op == "quantize":
        n = c["rows"] * c["cols"]
        # the float values that the codes stand for are not counted: the operator's result is the codes
        return dict(bytes=n * (SIZE[c["dtype"]] + 1) + 4 * c["rows"] + (4 * c["cols"] if c["norm"] else 0), flops=4 * n)
    if op == "matmul":
        m, n, k = c["m"], c["n"], c["k"]
        return dict(bytes=m * k + n * k + m * n * SIZE[c["out"]] + 4 * (m + n), flops=2 * m * n * k)
    if op == "lmhead":
        r, h, v = c["rows"], c["hidden"], c["vocab"]
        return dict(bytes=v * h + 4 * v + 4 * r * h + 4 * h + 4 * r * v, flops=2 * r * h * v)
    if op == "select":
        rows = c["batch"] if c["first"] else c["batch"] * c["beams"] - int(c["finished"] * c["batch"] * c["beams"])
        rows = max(1, rows)
        per = c["vocab"] * SIZE[c["dtype"]] + (4 * ((c["vocab"] + 31) // 32) if c["allowed"] < 1 else 0)
        return dict(bytes=rows * per + 12 * c["batch"] * c["k"] + 9 * c["batch"] * c["beams"], flops=4 * rows * c["vocab"])
    run_bytes = c["length"] * c["dim"] * SIZE[c["dtype"]] * c["heads"]
    return dict(bytes=c["tensors"] * c["batch"] * run_bytes * (c["moved"] + min(_sources(c), c["moved"])), flops=0)


# ---- inputs ------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _codes(g, rows, cols):
    """int8 codes as symmetric quantisation leaves them: a normal row's largest value is about 4 sigma.
    Rows start on multiples of 16 bytes."""
    ld = (cols + 15) // 16 * 16
    q = torch.empty(rows, ld, dtype=torch.int8, device="cuda")
    for at in range(0, rows, 16384):
        part = q[at:at + 16384]
        part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 31).round_().clamp_(-127, 127))
    return q[:, :cols]


def _scales(g, n, size):
    return (torch.rand(n, generator=g, device="cuda") + 0.5) * size


def _pack(allow):
    rows, width = allow.shape
    words = (allow.view(rows, width // 32, 32).to(torch.int64) << torch.arange(32, device="cuda")).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def prepare(case, seed):
    c, op, g = case, case["op"], _gen(seed)
    s = dict(case=case)
    if op == "quantize":
        x = _normal(g, c["rows"], c["cols"])
        x *= torch.exp(0.5 * _normal(g, c["rows"], 1))  # rows of different sizes
        s["x"] = x.to(DTYPES[c["dtype"]])
        if c["norm"]:
            s["w"] = 1 + 0.2 * _normal(g, c["cols"])
    elif op == "matmul":
        s["a"], s["sa"] = _codes(g, c["m"], c["k"]), _scales(g, c["m"], 0.03)
        s["b"], s["sb"] = _codes(g, c["n"], c["k"]), _scales(g, c["n"], 0.001)
    elif op == "lmhead":
        s["h"] = 3 * _normal(g, c["rows"], c["hidden"])
        s["w"] = 0.2 * _normal(g, c["hidden"]) + (0 if c["add_one"] else 1)
        # logits of a standard deviation of about 3
        s["wq"], s["sw"] = _codes(g, c["vocab"], c["hidden"]), _scales(g, c["vocab"], 3 / 31 / c["hidden"] ** 0.5)
    elif op == "select":
        B, K, V = c["batch"], c["beams"], c["vocab"]
        x = torch.empty(B * K, V, dtype=DTYPES[c["dtype"]], device="cuda")
        for b in range(B):  # beams of one sequence agree in part; 20 ids stand out
            r = 1.5 * _normal(g, 1, V) + _normal(g, K, V)
            r[:, torch.randint(0, V, (20,), generator=g, device="cuda")] += 8
            x[b * K:(b + 1) * K] = r
        s["x"] = x
        s["scores"] = -4 * torch.rand(B, K, generator=g, device="cuda").cumsum(1)
        if c["first"]:  # the first step: one live beam
            s["scores"][:, 1:] = -math.inf
        s["mask"] = s["finished"] = s["lengths"] = None
        if c["allowed"] < 1:
            W = (V + 31) // 32
            allow = torch.rand(B * K, 32 * W, generator=g, device="cuda") < c["allowed"]
            allow[:, V:] = False
            s["mask"] = _pack(allow)
        if c["finished"] > 0:
            n = int(c["finished"] * B * K)
            done = torch.zeros(B * K, dtype=torch.uint8, device="cuda")
            done[torch.randperm(B * K, generator=g, device="cuda")[:n]] = 1
            s["finished"] = done.view(B, K)
        if c["alpha"] > 0:
            s["lengths"] = torch.randint(5, 40, (B, K), generator=g, device="cuda", dtype=torch.int32)
        s["eos"] = 2
    else:
        B, K = c["batch"], c["beams"]
        s["states"] = []
        for _ in range(c["tensors"]):
            shape = (B * K, c["heads"], c["cap"], c["dim"])
            if c["dtype"] == "i32":
                t = torch.randint(0, 128256, shape, generator=g, device="cuda", dtype=torch.int32)
            else:
                t = _normal(g, *shape).to(DTYPES[c["dtype"]])
            s["states"].append(t[:, :, :c["length"]])
        own_beam = torch.arange(K, device="cuda").expand(B, K)
        step = torch.randint(1, K, (B, K), generator=g, device="cuda")
        chosen = torch.rand(B, K, generator=g, device="cuda").argsort(1) < c["moved"]
        s["parents"] = torch.where(chosen, (own_beam + step) % K, own_beam).to(torch.int32)
    torch.cuda.synchronize()
    return s


# ---- the plain forms ---------------------------------------------------------------------------

def _plain_codes(x, norm, w, add_one):
    """Codes in 64 bits: which of two neighbours a value next to a border rounds to depends on it."""
    y = x.double()
    if norm:
        eps = float(torch.tensor(EPS, dtype=F32))
        y = y / (y.square().mean(1, keepdim=True) + eps).sqrt()
        if w is not None:
            y = y * (w.double() + (1 if add_one else 0))
    scale = (y.abs().amax(1) / 127).float()
    q = torch.where(scale[:, None] > 0, (y / scale.double()[:, None]).round(), torch.zeros_like(y))
    return q, scale


def _plain_product(a, sa, b, sb):
    return (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()[None, :]


def _plain_select(s):
    c, x = s["case"], s["x"]
    B, K, V, k = c["batch"], c["beams"], c["vocab"], c["k"]
    x = x.float()
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = torch.where(bits.view(B * K, -1)[:, :V] > 0, x, x.new_tensor(-math.inf))
    top = x.amax(1, keepdim=True)
    at = torch.where(top > -math.inf, top, torch.zeros_like(top))
    lse = (at.double() + (x - at).double().exp().sum(1, keepdim=True).log()).view(B, K, 1)
    # the k best of each row, by logit and then by id: keys of 64 bits, no two alike
    low = x.view(torch.int32)
    key = torch.where(low >= 0, low, low ^ 0x7FFFFFFF).to(torch.int64) << 32
    key += (2 ** 31 - 1) - torch.arange(V, device=x.device)
    ids = key.topk(min(k, V), dim=1).indices
    cum = s["scores"].double()[:, :, None] + (x.gather(1, ids).double().view(B, K, -1) - lse)
    tokens = ids.view(B, K, -1)
    if s["finished"] is not None:  # an ended beam goes on as it is, once
        first = torch.arange(cum.shape[2], device=x.device) == 0
        kept = torch.where(first, s["scores"].double()[:, :, None], torch.full_like(cum, -math.inf))
        done = s["finished"].bool()[:, :, None]
        cum = torch.where(done, kept, cum)
        tokens = torch.where(done, torch.full_like(tokens, s["eos"]), tokens)
    cum = torch.where(cum > -math.inf, cum, torch.full_like(cum, -math.inf))  # NaN: nothing to choose
    rank = cum
    if c["alpha"] > 0:
        n = s["lengths"].double() + (1 if s["finished"] is None else 1 - s["finished"].double())
        rank = cum / n.pow(c["alpha"])[:, :, None]
    best = rank.reshape(B, -1).sort(dim=1, descending=True, stable=True).indices[:, :k]
    score = cum.reshape(B, -1).gather(1, best)
    parent = best // cum.shape[2]
    token = tokens.reshape(B, -1).gather(1, best)
    none = score == -math.inf
    short = k - best.shape[1]
    out = [score.float(), parent.masked_fill(none, -1).int(), token.masked_fill(none, -1).int()]
    if short > 0:
        out = [torch.cat([o, o.new_full((B, short), f)], 1) for o, f in zip(out, (-math.inf, -1, -1))]
    return tuple(out)


def _plain_reorder(s):
    p, K = s["parents"], s["case"]["beams"]
    rows = (torch.arange(p.shape[0], device=p.device)[:, None] * K + p).reshape(-1)
    for t in s["states"]:
        t.copy_(t.index_select(0, rows))
    return s["states"]


def run(state):
    s = state
    c, op = s["case"], s["case"]["op"]
    if own:
        from diskllm_b200 import capi

        if op == "quantize":
            q, scale = capi.quantize_rows_i8(s["x"], norm=c["norm"], norm_w=s.get("w"), eps=EPS)
            return torch.mul(q, scale[:, None]), scale
        if op == "matmul":
            return capi.matmul_i8(s["a"], s["sa"], s["b"], s["sb"], out_dtype=DTYPES[c["out"]])
        if op == "lmhead":
            return capi.lmhead_logits_i8(s["h"], s["wq"], s["sw"], norm_w=s["w"], eps=EPS, add_one=c["add_one"],
                                         softcap=c["softcap"])
        if op == "select":
            return capi.beam_select(s["x"], s["scores"], c["k"], mask=s["mask"], finished=s["finished"],
                                    eos=s["eos"], lengths=s["lengths"], length_penalty=c["alpha"])
        capi.beam_reorder(s["states"], s["parents"])
        return s["states"]
    if op == "quantize":
        q, scale = _plain_codes(s["x"], c["norm"], s.get("w"), False)
        return torch.mul(q.to(torch.int8), scale[:, None]), scale
    if op == "matmul":
        return _plain_product(s["a"], s["sa"], s["b"], s["sb"]).to(DTYPES[c["out"]])
    if op == "lmhead":
        q, scale = _plain_codes(s["h"], True, s["w"], c["add_one"])
        y = _plain_product(q, scale, s["wq"], s["sw"])
        return (c["softcap"] * (y / c["softcap"]).tanh() if c["softcap"] > 0 else y).float()
    if op == "select":
        return _plain_select(s)
    return _plain_reorder(s)


# ---- the definitions in 64 bits ----------------------------------------------------------------

def _exact_codes(x, norm, w, add_one):
    """(codes, scales): code = the integer next to value / scale, ties to even; scale = largest / 127,
    a number of 32 bits, since that is what the operator gives out."""
    codes, scales = [], []
    for row in x.split(max(1, (1 << 26) // x.shape[1])):
        v = row.to(torch.float64)
        if norm:
            n = v.shape[1]
            rms = torch.sqrt((v * v).sum(1) / n + float(torch.tensor(EPS, dtype=F32)))
            gain = torch.ones(n, dtype=torch.float64, device=v.device) if w is None else w.to(torch.float64)
            v = v * (gain + 1.0 if add_one else gain) / rms[:, None]
        sc = (torch.maximum(v.amax(1), -v.amin(1)) / 127.0).to(F32).to(torch.float64)
        r = v / torch.where(sc > 0, sc, torch.ones_like(sc))[:, None]
        low = torch.floor(r)
        up = (r - low > 0.5) | ((r - low == 0.5) & (torch.remainder(low, 2) == 1))
        codes.append((low + up.to(torch.float64)).to(torch.int8))
        scales.append(sc)
    return torch.cat(codes), torch.cat(scales)


def _exact_product(a, sa, b, sb):
    """Sums of int8 products: pieces of 512 terms are whole numbers under 2^24, exact in 32 bits."""
    total = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device=a.device)
    for at in range(0, a.shape[1], 512):
        total += a[:, at:at + 512].to(F32) @ b[:, at:at + 512].to(F32).T
    return sa.to(torch.float64)[:, None] * (total * sb.to(torch.float64))


def _exact_select(s):
    c = s["case"]
    B, K, V = c["batch"], c["beams"], c["vocab"]
    out = torch.full((B, c["k"]), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(B):
        z = s["x"][b * K:(b + 1) * K].to(torch.float64)
        if s["mask"] is not None:
            words = s["mask"][b * K:(b + 1) * K].to(torch.int64)
            i = torch.arange(V, device=z.device)
            z = z.masked_fill(((words[:, i // 32] >> (i % 32)) & 1) == 0, -math.inf)
        cum = z - torch.logsumexp(z, 1, keepdim=True) + s["scores"][b].to(torch.float64)[:, None]
        length = torch.ones(K, dtype=torch.float64, device=z.device)
        if c["alpha"] > 0:
            length = length + s["lengths"][b]
        if s["finished"] is not None:
            f = s["finished"][b].bool()
            cum[f] = -math.inf
            cum[f, s["eos"]] = s["scores"][b].to(torch.float64)[f]
            length = torch.where(f, length - 1, length) if c["alpha"] > 0 else length
        cum = torch.nan_to_num(cum, nan=-math.inf, neginf=-math.inf)
        rank = cum / length[:, None] ** c["alpha"] if c["alpha"] > 0 else cum
        n = min(c["k"], K * V)
        out[b, :n] = cum.flatten()[torch.topk(rank.flatten(), n).indices]
    return out, None, None


def exact(case, seed):
    s, c, op = prepare(case, seed), case, case["op"]
    if op == "quantize":
        q, scale = _exact_codes(s["x"], c["norm"], s.get("w"), False)
        return q.to(torch.float64) * scale[:, None], scale
    if op == "matmul":
        return _exact_product(s["a"], s["sa"], s["b"], s["sb"])
    if op == "lmhead":
        q, scale = _exact_codes(s["h"], True, s["w"], c["add_one"])
        y = _exact_product(q, scale, s["wq"], s["sw"])
        return torch.tanh(y / c["softcap"]) * c["softcap"] if c["softcap"] > 0 else y
    if op == "select":
        return _exact_select(s)
    if c["dtype"] == "i32":
        return None  # whole numbers
    K = c["beams"]
    new = []
    for t in s["states"]:
        by_beam = t.reshape(c["batch"], K, *t.shape[1:])
        moved = [torch.stack([by_beam[b, j] for j in s["parents"][b].tolist()]) for b in range(c["batch"])]
        new.append(torch.cat(moved).to(torch.float64))
    return new
