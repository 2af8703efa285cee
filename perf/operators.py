"""The measured cases of the low-precision attention layer: norm to 8 bits, the 4-bit K/V cache, and attention over that cache.

Four operators: ``norm`` (RMSNorm, with or without the residual's addition, to e4m3 rows with one scale each), ``cache`` (K/V rows into
a 4-bit cache and back), ``questions`` (packed questions over one shared 4-bit state and their own keys, or a causal prompt) and
``decode`` (the newest tokens of many sequences, each over its own stretch of a 4-bit cache).

A cache row holds, for every K/V head, head_dim e2m1 codes (two per byte, the even one in the low nibble) and one e4m3 scale for each
16 of them; a value is code * scale.
"""
import ctypes
import math
import random

import torch

own = False

EPS = 1e-6
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # between neighbouring e2m1 magnitudes; a tie goes up
DTYPES = {"f32": (0, torch.float32, 4), "bf16": (1, torch.bfloat16, 2)}


# ---- the cases ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the norm of one new token, hidden 5120: what every layer of a single-token step pays
        {"name": "norm_token", "op": "norm", "rows": 1, "cols": 5120, "dtype": "bf16", "add": True},
        # an f32 engine's rows inside a wider matrix, an odd width
        {"name": "norm_f32_odd", "op": "norm", "rows": 301, "cols": 775, "dtype": "f32", "add": False},
        # one cold request: a state of 2048 tokens and 64 questions (6835 tokens) in one pass
        {"name": "norm_request", "op": "norm", "rows": 8883, "cols": 5120, "dtype": "bf16", "add": True},
        # the K/V of one new token of each of 64 sequences, to scattered rows of the cache
        {"name": "cache_tokens", "op": "cache", "rows": 64, "kv": 4, "hd": 256, "dtype": "bf16"},
        # the tiny f32 model's single head of 64
        {"name": "cache_f32_small", "op": "cache", "rows": 1001, "kv": 1, "hd": 64, "dtype": "f32"},
        # a state of 16384 tokens taken from the fused q/k/v projection
        {"name": "cache_state", "op": "cache", "rows": 16384, "kv": 4, "hd": 256, "dtype": "bf16"},
        # one question of 16 tokens over a state of 4096: the smallest request, latency counts
        {"name": "question_one", "op": "questions", "B": 1, "lo": 16, "hi": 16, "S": 4096, "heads": 24, "kv": 4, "hd": 256, "causal": False, "gate": True},
        # 64 questions of about 107 tokens over a state of 2048
        {"name": "questions_64", "op": "questions", "B": 64, "lo": 64, "hi": 150, "S": 2048, "heads": 24, "kv": 4, "hd": 256, "causal": False, "gate": True},
        # five prompts packed behind each other, causal, grouped heads of 128, nothing cached yet
        {"name": "prompt_causal", "op": "questions", "B": 5, "lo": 700, "hi": 2048, "S": 0, "heads": 16, "kv": 2, "hd": 128, "causal": True, "gate": False},
        # one sequence, one token: the latency of a step
        {"name": "decode_one", "op": "decode", "B": 1, "L": 1, "lo": 2048, "hi": 2048, "heads": 24, "kv": 4, "hd": 256},
        # 64 sequences of very different lengths, one token each: the throughput of a step
        {"name": "decode_64", "op": "decode", "B": 64, "L": 1, "lo": 1024, "hi": 16384, "heads": 24, "kv": 4, "hd": 256},
        # four drafted tokens a sequence, checked at once
        {"name": "decode_drafts", "op": "decode", "B": 9, "L": 4, "lo": 500, "hi": 8192, "heads": 16, "kv": 2, "hd": 128},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = ((24, 4, 256), (4, 1, 64), (16, 2, 128), (8, 8, 128), (12, 2, 64), (16, 1, 128), (15, 3, 256))


def draw(rng):
    op = rng.choice(("norm", "cache", "questions", "decode"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    half = 2 if dtype == "f32" else 1
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 8883 // half), "cols": _log(rng, 33, 5120), "dtype": dtype, "add": rng.random() < 0.6}
    heads, kv, hd = rng.choice(HEADS)
    if op == "cache":
        return {"op": op, "rows": _log(rng, 1, 16384 // half), "kv": kv, "hd": hd, "dtype": dtype}
    if op == "questions":
        if rng.random() < 0.3:
            lo = _log(rng, 1, 600)
            return {"op": op, "B": rng.randint(1, 5), "lo": lo, "hi": lo + _log(rng, 1, 1400), "S": rng.choice((0, _log(rng, 1, 2048))), "heads": heads, "kv": kv, "hd": hd,
                    "causal": True, "gate": rng.random() < 0.5}
        lo, S = _log(rng, 1, 64), _log(rng, 1, 16384)
        return {"op": op, "B": _log(rng, 1, min(64, max(1, 120000 // S))), "lo": lo, "hi": lo + _log(rng, 1, 80), "S": S, "heads": heads, "kv": kv, "hd": hd,
                "causal": rng.random() < 0.3, "gate": rng.random() < 0.5}
    lo = _log(rng, 1, 2000)
    return {"op": op, "B": _log(rng, 1, 64), "L": rng.choice((1, 1, 2, 4)), "lo": lo, "hi": lo + _log(rng, 1, 12000), "heads": heads, "kv": kv, "hd": hd}


def _lens(case):
    """The sequences' lengths (tokens of a question, cached rows of a sequence): part of the case, not of its inputs."""
    r = random.Random("%d %d %d" % (case["B"], case["lo"], case["hi"]))
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
def _cu(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _codes(g, rows, kv, hd):
    """A cache of values with an rms of about one: uniform codes, scales of a factor of four."""
    codes = torch.randint(0, 256, (rows, kv, hd // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = (torch.rand((rows, kv, hd // 16), device="cuda", generator=g) * 0.375 + 0.125).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, by=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * by).to(dtype)

    s = dict(case)
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        _, t, _ = DTYPES[case["dtype"]]
        # a residual stream: a few channels far larger than the others; the rows lie 64 elements apart from each other
        big = 1 + 30 * (torch.rand(cols + 64, device="cuda", generator=g) < 0.01)
        s["x"] = (normal(rows, cols + 64, dtype=torch.float32) * big).to(t)[:, :cols]
        s["mix"] = normal(rows, cols, dtype=t) if case["add"] else None
        s["w"] = normal(cols, dtype=t, by=0.1)
        s["residual"] = torch.empty(rows, cols, dtype=t, device="cuda")
        s["q"] = torch.empty(rows, cols, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty(rows, dtype=torch.float32, device="cuda")
    elif case["op"] == "cache":
        rows, kv, hd = case["rows"], case["kv"], case["hd"]
        _, t, _ = DTYPES[case["dtype"]]
        wide = normal(rows, 4 * kv * hd, dtype=t)  # a fused projection: two parts of q, then k, then v
        s["k"], s["v"] = wide[:, 2 * kv * hd:3 * kv * hd], wide[:, 3 * kv * hd:]
        s["cache_rows"] = rows + 100
        s["slots"] = torch.randperm(s["cache_rows"], device="cuda", generator=g)[:rows].contiguous()
        for n, width in (("k_codes", hd // 2), ("k_scales", hd // 16), ("v_codes", hd // 2), ("v_scales", hd // 16)):
            s[n] = torch.zeros(s["cache_rows"], kv, width, dtype=torch.uint8, device="cuda")
        s["k_out"], s["v_out"] = (torch.empty(rows, kv, hd, dtype=t, device="cuda") for _ in range(2))
    elif case["op"] == "questions":
        heads, kv, hd, lens = case["heads"], case["kv"], case["hd"], _lens(case)
        T = sum(lens)
        s["T"], s["longest"] = T, max(lens)
        s["q"] = normal(T, heads, hd, by=1.5)
        s["k"], s["v"] = (normal(T, kv * hd + 64)[:, :kv * hd] for _ in range(2))  # rows of a wider matrix
        s["qg"] = normal(T, heads, 2 * hd) if case["gate"] else None
        s["k_codes"], s["k_scales"] = _codes(g, case["S"], kv, hd)
        s["v_codes"], s["v_scales"] = _codes(g, case["S"], kv, hd)
        s["cu"] = _cu(lens)
        s["out"] = torch.empty(T, heads, hd, dtype=torch.bfloat16, device="cuda")
        s["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    else:
        heads, kv, hd, lens = case["heads"], case["kv"], case["hd"], _lens(case)
        T = case["B"] * case["L"]
        s["T"], s["longest"] = T, max(lens)
        order = list(range(case["B"]))
        random.Random(seed).shuffle(order)  # where each sequence lies in the pool, a gap behind each
        start, at = [0] * case["B"], 3
        for b in order:
            start[b], at = at, at + lens[b] + 5
        s["pool"] = at
        s["k_codes"], s["k_scales"] = _codes(g, at, kv, hd)
        s["v_codes"], s["v_scales"] = _codes(g, at, kv, hd)
        s["start"] = torch.tensor(start, dtype=torch.int64, device="cuda")
        s["len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["cu"] = _cu([case["L"]] * case["B"])
        s["q"] = normal(T, heads, hd, by=1.5)
        s["out"] = torch.empty(T, heads, hd, dtype=torch.bfloat16, device="cuda")
        s["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------------------
def _table(device):
    return torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=device)


def _values(codes, scales):
    """[rows, kv, hd / 2] codes and [rows, kv, hd / 16] scales -> [rows, kv, hd] in f32."""
    rows, kv, half = codes.shape
    pair = torch.stack((codes & 15, codes >> 4), -1).long()
    v = _table(codes.device)[pair].reshape(rows, kv, half // 8, 16)
    return (v * scales.view(torch.float8_e4m3fn).float()[..., None]).reshape(rows, kv, 2 * half)


def _encode(x):
    """[rows, kv, hd] -> codes and scales."""
    rows, kv, hd = x.shape
    v = x.float().reshape(rows, kv, hd // 16, 16)
    sf = torch.clamp(v.abs().amax(-1) / 6, min=1e-10).clamp(max=448).to(torch.float8_e4m3fn)
    y = v / sf.float()[..., None]
    code = torch.bucketize(y.abs(), torch.tensor(BORDERS, device=x.device), right=True) + 8 * (y < 0)
    code = code.to(torch.uint8).reshape(rows, kv, hd // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), sf.view(torch.uint8)


def _plain_norm(s):
    x = s["x"].float()
    if s["add"]:
        s["residual"].copy_(x + s["mix"].float())
        x = s["residual"].float()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + s["w"].float())
    scale = torch.clamp(y.abs().amax(-1), min=1e-10) / 448
    q = (y / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return (q, scale, s["residual"]) if s["add"] else (q, scale)


def _plain_cache(s):
    rows, kv, hd = s["rows"], s["kv"], s["hd"]
    for n in "kv":
        codes, scales = _encode(s[n].reshape(rows, kv, hd))
        s[n + "_codes"][s["slots"]], s[n + "_scales"][s["slots"]] = codes, scales
        s[n + "_out"].copy_(_values(s[n + "_codes"][s["slots"]], s[n + "_scales"][s["slots"]]))
    return s["k_out"], s["v_out"]


def _plain_questions(s):
    T, B, S, heads, kv, hd = s["T"], s["B"], s["S"], s["heads"], s["kv"], s["hd"]
    L, G = s["longest"], heads // kv
    cu = s["cu"].long()
    at = torch.arange(L, device="cuda")
    inside = at[None] < (cu[1:] - cu[:-1])[:, None]  # [B, L]
    index = torch.where(inside, cu[:-1, None] + at, 0)
    q = s["q"].float().reshape(T, kv, G, hd) / math.sqrt(hd)
    k, v = (s[n].float().reshape(T, kv, hd) for n in "kv")
    # own keys, every sequence padded to the longest
    qp, kp = q[index], k[index]
    vp = torch.where(inside[:, :, None, None], v[index], 0.0)
    seen = inside[:, None, :]
    if s["causal"]:
        seen = seen & (at[None, :, None] >= at[None, None, :])
    scores = torch.einsum("bikgd,bjkd->bkgij", qp, kp).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1)  # [B, kv, G, L]; a padded row sees nothing of its own: its answers are not taken
    if S:
        ks, vs = _values(s["k_codes"], s["k_scales"]), _values(s["v_codes"], s["v_scales"])
        state = torch.einsum("tkgd,jkd->tkgj", q, ks)
        top = torch.maximum(top, state.amax(-1)[index].permute(0, 2, 3, 1))
    top = top.clamp(min=-1e30)
    p = torch.exp(scores - top[..., None])
    sums = p.sum(-1)[..., None].permute(0, 3, 1, 2, 4)[inside]  # [T, kv, G, 1]: the packed rows in order
    out = torch.einsum("bkgij,bjkd->bikgd", p, vp)[inside]
    if S:
        p = torch.exp(state - top.permute(0, 3, 1, 2)[inside][..., None])
        sums = sums + p.sum(-1, keepdim=True)
        out = out + torch.einsum("tkgj,jkd->tkgd", p, vs)
    out = (out / sums).reshape(T, heads, hd)
    if s["gate"]:
        out = out * torch.sigmoid(s["qg"].float()[:, :, hd:])
    return out.to(torch.bfloat16)


def _plain_decode(s):
    B, L, heads, kv, hd, T = s["B"], s["L"], s["heads"], s["kv"], s["hd"], s["T"]
    at = torch.arange(s["longest"], device="cuda")
    n = s["len"].long()
    inside = at[None] < n[:, None]
    index = torch.where(inside, s["start"][:, None] + at, 0)
    k = _values(s["k_codes"], s["k_scales"])[index]  # [B, longest, kv, hd]
    q = s["q"].float().reshape(B, L, kv, heads // kv, hd) / math.sqrt(hd)
    scores = torch.einsum("bikgd,bjkd->bkgij", q, k)
    del k
    last = n[:, None] - L + torch.arange(L, device="cuda")  # the last row that each token sees; none where it is negative
    seen = at[None, None] <= last[:, :, None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    v = torch.where(inside[:, :, None, None], _values(s["v_codes"], s["v_scales"])[index], 0.0)
    out = torch.einsum("bkgij,bjkd->bikgd", p, v)
    out = out / p.sum(-1).permute(0, 3, 1, 2)[..., None].clamp(min=1e-30)
    return out.reshape(T, heads, hd).to(torch.bfloat16)


# ---- the framework's calls ------------------------------------------------------------------------------------------------------
def _call(name, *args):
    from decidra_b200 import _lib

    args = [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]
    rc = getattr(_lib.load(), name)(*args)
    if rc:
        raise RuntimeError("%s returned %d" % (name, rc))


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _workspace(s, name, *args):
    """A workspace of the size that the library asks for, kept with the state as a program keeps it with its engine."""
    if "workspace" not in s:
        from decidra_b200 import _lib

        s["workspace"] = torch.empty(max(1, getattr(_lib.load(), name)(*args)), dtype=torch.uint8, device="cuda")
    return s["workspace"]


def _own_norm(s):
    x, code = s["x"], DTYPES[s["dtype"]][0]
    rows, cols = x.shape
    if s["add"]:
        _call("dcd_k_add_rmsnorm_fp8", x, x.stride(0), s["mix"], s["mix"].stride(0), s["w"], s["residual"], s["q"], s["scales"], rows, cols, EPS, 1, 1.0, 0, code, _stream())
        return s["q"].view(torch.float8_e4m3fn), s["scales"], s["residual"]
    _call("dcd_k_rmsnorm_fp8", x, x.stride(0), s["w"], s["q"], s["scales"], rows, cols, EPS, 1, 1.0, 0, code, _stream())
    return s["q"].view(torch.float8_e4m3fn), s["scales"]


def _own_cache(s):
    code, cache = DTYPES[s["dtype"]][0], (s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], s["cache_rows"])
    _call("dcd_k_kv4_write", s["k"], s["k"].stride(0), s["v"], s["v"].stride(0), s["slots"], *cache, s["rows"], s["kv"], s["hd"], code, None, _stream())
    _call("dcd_k_kv4_read", *cache, s["slots"], s["k_out"], s["v_out"], s["rows"], s["kv"], s["hd"], code, None, _stream())
    return s["k_out"], s["v_out"]


def _own_questions(s):
    shape = (s["heads"], s["kv"], s["hd"])
    ws = _workspace(s, "dcd_k_attention_kv4_workspace", s["B"], s["T"], s["S"], *shape)
    state = [s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"]] if s["S"] else [None] * 4
    _call("dcd_k_attention_kv4", s["q"], s["heads"] * s["hd"], s["k"], s["k"].stride(0), s["v"], s["v"].stride(0), *state, s["S"], s["qg"], 2 * s["heads"] * s["hd"],
          s["out"], s["cu"], s["B"], s["T"], *shape, int(s["causal"]), ws, ws.numel(), s["err"], _stream())
    return s["out"]


def _own_decode(s):
    shape = (s["heads"], s["kv"], s["hd"])
    ws = _workspace(s, "dcd_k_attention_kv4_decode_workspace", s["B"], s["T"], s["longest"], *shape)
    _call("dcd_k_attention_kv4_decode", s["q"], s["heads"] * s["hd"], s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], s["pool"], s["start"], s["len"],
          s["longest"], None, 0, s["out"], s["cu"], s["B"], s["T"], *shape, ws, ws.numel(), s["err"], _stream())
    return s["out"]


def run(state):
    op = state["op"]
    if own:
        return (_own_norm if op == "norm" else _own_cache if op == "cache" else _own_questions if op == "questions" else _own_decode)(state)
    return (_plain_norm if op == "norm" else _plain_cache if op == "cache" else _plain_questions if op == "questions" else _plain_decode)(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        n, size = case["rows"] * case["cols"], DTYPES[case["dtype"]][2]
        return {"bytes": n * (size * (3 if case["add"] else 1) + 1) + 4 * case["rows"] + size * case["cols"], "flops": 8 * n}
    if case["op"] == "cache":  # written and read back
        n, size = 2 * case["rows"] * case["kv"] * case["hd"], DTYPES[case["dtype"]][2]
        return {"bytes": n * (2 * size + 2 * 0.5625) + 16 * case["rows"], "flops": 4 * n}
    heads, kv, hd, lens = case["heads"], case["kv"], case["hd"], _lens(case)
    if case["op"] == "questions":
        T, S = sum(lens), case["S"]
        pairs = sum(n * S + (n * (n + 1) // 2 if case["causal"] else n * n) for n in lens)
        return {"bytes": 2 * T * heads * hd * (3 if case["gate"] else 2) + 4 * T * kv * hd + 1.125 * S * kv * hd, "flops": 4 * heads * hd * pairs}
    L = case["L"]
    pairs = sum(max(0, n - L + i + 1) for n in lens for i in range(L))
    return {"bytes": 4 * case["B"] * L * heads * hd + 1.125 * sum(lens) * kv * hd, "flops": 4 * heads * hd * pairs}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------
def _exact_values(codes, scales):
    mag = torch.tensor(E2M1, dtype=torch.float64, device=codes.device)
    rows, kv, half = codes.shape
    out = torch.empty(rows, kv, half, 2, dtype=torch.float64, device=codes.device)
    for i in range(2):
        c = ((codes >> (4 * i)) & 15).long()
        out[..., i] = mag[c & 7] * (1 - 2 * (c >> 3))
    return out.reshape(rows, kv, 2 * half) * scales.view(torch.float8_e4m3fn).double().repeat_interleave(16, -1)


def _exact_e4m3(y):
    """The nearest e4m3 value, ties to even, of |y| <= 448."""
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp(min=-6) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def _exact_attention(q, k, v, seen, gate):
    """q [n, heads, hd], k and v [m, kv, hd], seen [n, m]; rows that see nothing give 0."""
    n, heads, hd = q.shape
    kv = k.shape[1]
    out = torch.zeros_like(q)
    for h in range(heads):
        a = (q[:, h] @ k[:, h // (heads // kv)].T / math.sqrt(hd)).masked_fill(~seen, -math.inf)
        p = torch.nan_to_num(torch.softmax(a, -1), nan=0.0)
        out[:, h] = p @ v[:, h // (heads // kv)]
    return out if gate is None else out / (1 + torch.exp(-gate))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        r = s["x"].double()
        if case["add"]:
            total = r + s["mix"].double()
            r = total.to(s["x"].dtype).double()  # the stored sum is what is normalised
        y = r * torch.rsqrt(r.square().mean(1, keepdim=True) + EPS) * (s["w"].double() + 1)
        scale = y.abs().amax(1).clamp(min=1e-10) / 448
        q = _exact_e4m3(y / scale[:, None])
        return (q, scale, total) if case["add"] else (q, scale)
    if case["op"] == "cache":
        got = []
        for n in "kv":
            x = s[n].double().reshape(-1, 16)
            sf = _exact_e4m3((x.abs().amax(1) / 6).clamp(min=1e-10))
            y = x / sf[:, None]
            m = sum((y.abs() >= b).double() * (E2M1[i + 1] - E2M1[i]) for i, b in enumerate(BORDERS))
            got.append((torch.where(y < 0, -m, m) * sf[:, None]).reshape(case["rows"], case["kv"], case["hd"]))
        return tuple(got)
    lens, hd = _lens(case), case["hd"]
    out = []
    if case["op"] == "questions":
        ks, vs = _exact_values(s["k_codes"], s["k_scales"]), _exact_values(s["v_codes"], s["v_scales"])
        at = 0
        for n in lens:
            rows = slice(at, at + n)
            k, v = (torch.cat((a, s[m][rows].double().reshape(n, case["kv"], hd))) for a, m in ((ks, "k"), (vs, "v")))
            seen = torch.ones(n, case["S"] + n, dtype=torch.bool, device="cuda")
            if case["causal"]:
                seen[:, case["S"]:] = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
            out.append(_exact_attention(s["q"][rows].double(), k, v, seen, s["qg"][rows, :, hd:].double() if case["gate"] else None))
            at += n
        return torch.cat(out)
    L = case["L"]
    for b, n in enumerate(lens):
        a = int(s["start"][b])
        k, v = (_exact_values(s[m + "_codes"][a:a + n], s[m + "_scales"][a:a + n]) for m in "kv")
        seen = torch.arange(n, device="cuda")[None] <= (n - L + torch.arange(L, device="cuda"))[:, None]
        out.append(_exact_attention(s["q"][b * L:(b + 1) * L].double(), k, v, seen, None))
    return torch.cat(out)
