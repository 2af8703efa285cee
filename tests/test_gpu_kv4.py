"""The low-precision attention layer's kernels on the GPU, through the C ABI: the norm to e4m3 rows, the 4-bit K/V cache, and the
attention over it in its question, prompt and new-token forms, each against a plain implementation in 64 bits."""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


@pytest.fixture(scope="module")
def G(dcd):
    import torch
    assert torch.cuda.is_available()
    import gpu_util
    return gpu_util


def gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=1, by=1.0):
    import torch
    return (torch.randn(shape, device="cuda", generator=g) * by).to(torch.bfloat16 if dtype else torch.float32)


def stream():
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


# ---------------------------------------------------------------------------------------------
# norm to e4m3 rows
# ---------------------------------------------------------------------------------------------
def norm_call(G, x, mix, w, cols, zc=1, clip=1.0, round_t=0, residual=None, eps=1e-6):
    import torch
    rows, dtype = x.shape[0], 0 if x.dtype == torch.float32 else 1
    q = torch.full((rows, cols), 0x55, dtype=torch.uint8, device="cuda")
    sc = torch.full((rows,), float("nan"), device="cuda")
    if mix is None:
        G.call("dcd_k_rmsnorm_fp8", x, x.stride(0), w, q, sc, rows, cols, eps, zc, clip, round_t, dtype, None)
        return q, sc, None
    res = torch.full((rows, cols), float("nan"), dtype=x.dtype, device="cuda") if residual is None else residual
    G.call("dcd_k_add_rmsnorm_fp8", x, x.stride(0), mix, mix.stride(0), w, res, q, sc, rows, cols, eps, zc, clip, round_t, dtype, None)
    return q, sc, res


def norm_check(x, mix, w, zc, clip, q, sc, res, eps=1e-6):
    import torch
    r = x.double()
    if mix is not None:
        r = r + mix.double()
        assert torch.equal(res, r.to(x.dtype))  # one rounded addition (f32: the sum of two f32 in f64 rounds to the same)
        r = res.double()
    y = r / torch.sqrt(r.square().mean(1, keepdim=True) + eps) * (w.double() + zc)
    s = (y.abs().amax(1) * clip).clamp(min=1e-10) / 448
    # the sum of squares: at most cols / 32 additions in a row a thread and ten across the block, each 2^-24, halved by the root, and
    # five more roundings behind it
    slack = (x.shape[1] / 32 + 10) * 2.0 ** -25 + 6 * 2.0 ** -24
    assert ((sc.double() - s).abs() <= slack * s).all()
    want = (y / s[:, None]).clamp(-448, 448)
    got = q.view(torch.float8_e4m3fn).double()
    # half a step: 2^-4 of the value, 2^-10 among the subnormals; and the slack twice (y and s)
    tol = torch.maximum(want.abs() * 2.0 ** -4, torch.full_like(want, 2.0 ** -10)) + 2 * slack * want.abs()
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,cols,pad", [(1, 5120, 0), (3, 64, 0), (37, 5120, 64), (5, 775, 64), (2, 1, 0), (7, 33, 1), (4, 8192, 8), (2, 8200, 0), (3, 20000, 3),
                                           (1, 40000, 0), (130, 688, 0)])
def test_norm_fp8(G, dtype, rows, cols, pad):
    g = gen(rows * 31 + cols)
    x = normal(g, rows, cols + pad, dtype=dtype, by=3.0)[:, :cols]
    mix = normal(g, rows, cols + 2 * pad, dtype=dtype)[:, :cols]
    w = normal(g, cols, dtype=dtype, by=0.1)
    for zc, clip in ((1, 1.0), (0, 0.5)):
        norm_check(x, None, w, zc, clip, *norm_call(G, x, None, w, cols, zc, clip))
        norm_check(x, mix, w, zc, clip, *norm_call(G, x, mix, w, cols, zc, clip))


def test_norm_fp8_rows_of_zeros_and_in_place(G):
    import torch
    g = gen(1)
    x, mix, w = normal(g, 6, 512), normal(g, 6, 512), normal(g, 512, by=0.1)
    x[2], mix[2] = 0, 0
    q, sc, res = norm_call(G, x, mix, w, 512)
    assert (q[2] & 0x7f == 0).all() and float(sc[2]) == np.float32(1e-10) / np.float32(448)
    for which in (0, 1):  # the residual over x, over mix
        a, b = x.clone(), mix.clone()
        q2, sc2, res2 = norm_call(G, a, b, w, 512, residual=(a, b)[which])
        assert torch.equal(q, q2) and torch.equal(sc, sc2) and torch.equal(res, res2)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,cols", [(1, 5120), (300, 5120), (3, 64), (2, 8192), (3, 8200), (5, 775), (4, 2500)])
def test_norm_fp8_rounded_form_has_the_bits_of_the_two_calls(G, dtype, rows, cols):
    import torch
    g = gen(rows + cols)
    x, mix, w = normal(g, rows, cols, dtype=dtype, by=2.0), normal(g, rows, cols, dtype=dtype), normal(g, cols, dtype=dtype, by=0.1)
    for add in (False, True):
        y, r = torch.empty_like(x), torch.empty_like(x)
        if add:
            G.call("dcd_k_add_rmsnorm", x, mix, w, r, y, rows, cols, C.c_float(1e-6), dtype, None)
        else:
            G.call("dcd_k_rmsnorm", x, w, y, rows, cols, C.c_float(1e-6), 1, dtype, None)
        q, sc = torch.empty((rows, cols), dtype=torch.uint8, device="cuda"), torch.empty(rows, device="cuda")
        G.call("dcd_k_quant_fp8_rows", y, C.c_size_t(cols), q, sc, rows, cols, C.c_float(1.0), dtype, None)
        q2, sc2, r2 = norm_call(G, x, mix if add else None, w, cols, round_t=1)
        assert torch.equal(q, q2) and torch.equal(sc, sc2) and (not add or torch.equal(r, r2))


# ---------------------------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------------------------
def new_cache(rows, kv, hd, fill=0x7F):
    """Every byte 0x7F: codes of -6 and scales of NaN, so that a row nobody wrote shows wherever it leaks."""
    import torch
    return [torch.full((rows, kv, hd // n), fill, dtype=torch.uint8, device="cuda") for n in (2, 16, 2, 16)]


def values(codes, scales):
    import torch
    t = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device="cuda")
    v = torch.stack((t[(codes & 15).long()], t[(codes >> 4).long()]), -1).reshape(*codes.shape[:2], -1)
    return v * scales.view(torch.float8_e4m3fn).double().repeat_interleave(16, -1)


def encoded(x):
    """The rule in 64 bits: the values that the cache then stands for."""
    import torch
    y = x.double().reshape(*x.shape[:-1], x.shape[-1] // 16, 16)
    sf = (y.abs().amax(-1) / 6).clamp(min=1e-10, max=448).to(torch.float8_e4m3fn).double()[..., None]
    z = y / sf
    m = sum((z.abs() >= b).double() * (E2M1[i + 1] - E2M1[i]) for i, b in enumerate(BORDERS))
    return (torch.where(z < 0, -m, m) * sf).reshape(x.shape)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,kv,hd,pad", [(1, 1, 64, 0), (7, 4, 256, 64), (33, 3, 128, 5), (130, 2, 64, 8), (1000, 4, 256, 0)])
def test_cache_write_and_read(G, dtype, rows, kv, hd, pad):
    import torch
    g = gen(rows + hd)
    k, v = (normal(g, rows, kv * hd + pad, dtype=dtype, by=by)[:, :kv * hd] for by in (2.0, 0.01))
    k[0, :16] = 0                       # a group of zeros
    v[-1, 16:32] = 1e-6                 # below the smallest scale: stands for zero
    k[-1, 32:48] = 5000.0               # above the largest value: saturates
    total = rows + 9
    slots = torch.randperm(total, device="cuda", generator=g)[:rows]
    slots[rows // 2] = -1               # left out
    cache = new_cache(total, kv, hd)
    before = [c.clone() for c in cache]
    err = G.devi([0])
    G.call("dcd_k_kv4_write", k, k.stride(0), v, v.stride(0), slots, *cache, total, rows, kv, hd, dtype, err, None)
    assert int(err.item()) == 0
    kept = slots >= 0
    for src, codes, scales in ((k, *cache[:2]), (v, *cache[2:])):
        got = values(codes, scales)[slots[kept]].reshape(-1, kv * hd)
        assert torch.equal(got, encoded(src[kept]))
    untouched = torch.ones(total, dtype=torch.bool, device="cuda")
    untouched[slots[kept]] = False
    for a, b in zip(cache, before):
        assert torch.equal(a[untouched], b[untouched])
    t = torch.float32 if dtype == 0 else torch.bfloat16
    ko, vo = (torch.full((rows, kv, hd), -7.0, dtype=t, device="cuda") for _ in range(2))
    G.call("dcd_k_kv4_read", *cache, total, slots, ko, vo, rows, kv, hd, dtype, err, None)
    for got, codes, scales in ((ko, *cache[:2]), (vo, *cache[2:])):
        assert torch.equal(got[kept].double(), values(codes, scales)[slots[kept]])  # exact in either type
        assert (got[~kept] == -7.0).all()
    assert int(err.item()) == 0


def test_cache_rows_in_order_and_the_bits_of_the_nvfp4_rows(G):
    import torch
    rows, kv, hd = 70, 4, 128
    g = gen(5)
    k, v = normal(g, rows, kv * hd), normal(g, rows, kv * hd, by=30.0)
    cache, err = new_cache(rows, kv, hd), G.devi([0])
    G.call("dcd_k_kv4_write", k, kv * hd, v, kv * hd, None, *cache, rows, rows, kv, hd, 1, err, None)
    for src, codes, scales in ((k, *cache[:2]), (v, *cache[2:])):
        c, s = torch.empty_like(codes), torch.empty_like(scales)
        G.call("dcd_k_nvfp4_quant_rows", src, C.c_size_t(kv * hd), C.c_float(1.0), c, s, rows, kv * hd, None)
        assert torch.equal(c, codes) and torch.equal(s, scales)
        out, two = torch.empty((rows, kv, hd), dtype=torch.bfloat16, device="cuda"), torch.empty((2, rows, kv, hd), dtype=torch.bfloat16, device="cuda")
        G.call("dcd_k_nvfp4_dequant_rows", codes, scales, out, rows, kv * hd, None)
        G.call("dcd_k_kv4_read", codes, scales, codes, scales, rows, None, two[0], two[1], rows, kv, hd, 1, err, None)
        assert torch.equal(out, two[0]) and torch.equal(out, two[1])


@pytest.mark.parametrize("dtype", [0, 1])
def test_cache_read_to_rows_of_16_byte_alignment(G, dtype):
    """What the interface asks for is 16 bytes: outputs, and an attention's workspace, that are not on 32."""
    import torch
    rows, kv, hd = 37, 2, 128
    cache = random_cache(gen(9), rows, kv, hd)
    t, skip = (torch.bfloat16, 8) if dtype else (torch.float32, 4)
    k, v = (torch.full((rows * kv * hd + 2 * skip,), -7.0, dtype=t, device="cuda") for _ in range(2))
    for shift_k, shift_v in ((skip, skip), (0, skip), (skip, 0)):
        a, b = k[shift_k:shift_k + rows * kv * hd], v[shift_v:shift_v + rows * kv * hd]
        G.call("dcd_k_kv4_read", *cache, rows, None, a, b, rows, kv, hd, dtype, None, None)
        torch.cuda.synchronize()
        assert torch.equal(a.double().reshape(rows, kv, hd), values(*cache[:2])) and torch.equal(b.double().reshape(rows, kv, hd), values(*cache[2:]))
    assert (k[-skip:] == -7.0).all() and (v[-skip:] == -7.0).all()


@pytest.mark.parametrize("form", ["questions", "prompts", "decode"])
def test_attention_operands_of_16_byte_alignment(G, form):
    import torch
    c = {"questions": lambda: Questions([40, 3], 5000, 16, 2, 128, False, True), "prompts": lambda: Questions([40, 300], 0, 24, 4, 256, True, True),
         "decode": lambda: Decode([5000, 40], 1, 24, 4, 256)}[form]()

    def shifted(x):  # the same values 16 bytes further on
        if x is None or not isinstance(x, torch.Tensor):
            return x
        skip = 16 // x.element_size()
        whole = torch.empty(x.untyped_storage().nbytes() // x.element_size() + skip, dtype=x.dtype, device="cuda")
        return torch.as_strided(whole, x.shape, x.stride(), skip + x.storage_offset()).copy_(x)

    c.launch(G)  # makes the workspace
    c.q, c.gate, c.out, c.cache = shifted(c.q), shifted(c.gate), shifted(c.out), [shifted(x) for x in c.cache]
    if form != "decode":
        c.k, c.v = shifted(c.k), shifted(c.v)
    c.ws = torch.full((c.ws.numel() + 16,), 0xFF, dtype=torch.uint8, device="cuda")[16:]
    c.out.fill_(-7.0)
    assert all(x.data_ptr() % 32 == 16 for x in (c.q, c.out, c.ws, *c.cache))
    c.launch(G)
    c.check()


def test_cache_values_that_are_not_finite_stay_in_their_group(G):
    import torch
    rows, kv, hd = 3, 1, 64
    k = normal(gen(6), rows, kv * hd)
    bad = k.clone()
    bad[1, 3], bad[1, 20] = float("nan"), float("inf")
    err = G.devi([0])
    a, b = new_cache(rows, kv, hd), new_cache(rows, kv, hd)
    G.call("dcd_k_kv4_write", k, hd, k, hd, None, *a, rows, rows, kv, hd, 1, err, None)
    G.call("dcd_k_kv4_write", bad, hd, bad, hd, None, *b, rows, rows, kv, hd, 1, err, None)
    va, vb = values(*a[:2])[:, 0], values(*b[:2])[:, 0]
    assert torch.isfinite(vb).all() and float(vb[1, 20]) == 2688.0
    assert torch.equal(va[:, 32:], vb[:, 32:]) and torch.equal(va[0], vb[0]) and torch.equal(va[2], vb[2])


def test_cache_slots_outside_set_the_error_word(G):
    import torch
    rows, kv, hd = 4, 2, 64
    k = normal(gen(7), rows, kv * hd)
    cache = new_cache(5, kv, hd)
    slots, err = torch.tensor([0, 5, 2 ** 40, 4], device="cuda"), G.devi([0])
    before = [c.clone() for c in cache]
    G.call("dcd_k_kv4_write", k, kv * hd, k, kv * hd, slots, *cache, 5, rows, kv, hd, 1, err, None)
    assert int(err.item()) == 7
    for c, b in zip(cache, before):
        assert torch.equal(c[1:4], b[1:4])
    assert torch.equal(values(*cache[:2])[[0, 4]].reshape(2, -1), encoded(k[[0, 3]]))
    out, err = torch.full((2, rows, kv, hd), -7.0, dtype=torch.bfloat16, device="cuda"), G.devi([0])
    G.call("dcd_k_kv4_read", *cache, 5, slots, out[0], out[1], rows, kv, hd, 1, err, None)
    assert int(err.item()) == 7 and (out[:, 1:3] == -7.0).all() and torch.isfinite(out).all()


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def random_cache(g, rows, kv, hd):
    import torch
    got = []
    for _ in range(2):
        got.append(torch.randint(0, 256, (rows, kv, hd // 2), dtype=torch.uint8, device="cuda", generator=g))
        got.append((torch.rand((rows, kv, hd // 16), device="cuda", generator=g) * 0.4 + 0.1).to(torch.float8_e4m3fn).view(torch.uint8))
    return got


def attend(q, k, v, seen):
    """64 bits: q [n, heads, hd], k and v [m, kv, hd], seen [n, m]. Returns the output and the sum of p |v| that bounds what rounding
    p costs; a row that sees nothing gives 0."""
    import torch
    rep = q.shape[1] // k.shape[1]
    k, v = (a.double().repeat_interleave(rep, 1) for a in (k, v))
    s = torch.einsum("ihd,jhd->hij", q.double(), k) / math.sqrt(q.shape[2])
    p = torch.nan_to_num(torch.softmax(s.masked_fill(~seen, -math.inf), -1), nan=0.0)
    return torch.einsum("hij,jhd->ihd", p, v), torch.einsum("hij,jhd->ihd", p, v.abs())


def close(got, want, spread, gate=None):
    """bf16 rounds the output by at most 2^-8 of it; p enters the second product rounded to 16 bits, at most 2^-8 of each p, and so
    does what its sum is made of: 2^-7 of sum p |v| together. The scores are f32 sums of head_dim exact products: 1e-3 covers their
    256 roundings of 2^-24 on sums of magnitudes below 64, and the exponentials'."""
    import torch
    if gate is not None:
        sg = torch.sigmoid(gate.double())
        want, spread = want * sg, spread * sg
    assert torch.isfinite(got).all()
    off = (got.double() - want).abs()
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -7 + 1e-3) * spread + 1e-30
    assert (off <= tol).all(), f"worst {float((off / tol).max()):.2f} of the tolerance at {[int(i) for i in np.unravel_index(int((off / tol).argmax()), off.shape)]}"


def cu_of(lens):
    return np.concatenate([[0], np.cumsum(lens)])


class Questions:
    """One call's operands. Rows of T behind the last sequence, the cache rows behind the state and the padding between the own rows
    hold NaN."""

    def __init__(self, lens, S, heads, kv, hd, causal, gate, seed=0, behind=3):
        import torch
        g = gen(seed + S + sum(lens) * 7 + hd)
        self.lens, self.S, self.heads, self.kv, self.hd, self.causal = lens, S, heads, kv, hd, causal
        self.n, self.T = sum(lens), sum(lens) + behind
        self.q = normal(g, self.T, heads, hd, by=1.5)
        wide = normal(g, self.T, 2 * kv * hd + 72)
        wide[self.n:] = float("nan")
        wide[:, kv * hd:kv * hd + 8] = float("nan")
        self.k, self.v = wide[:, :kv * hd], wide[:, kv * hd + 8:2 * kv * hd + 8]
        self.gate = normal(g, self.T, heads, 2 * hd) if gate else None
        rows = random_cache(g, S + 2, kv, hd)
        for i in (1, 3):
            rows[i][S:] = 0x7F
        self.cache = rows
        self.cu = torch.tensor(cu_of(lens), dtype=torch.int32, device="cuda")
        self.out = torch.full((self.T, heads, hd), -7.0, dtype=torch.bfloat16, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.ws = None

    def launch(self, G, st=None):
        import torch
        from decidra_b200 import _lib
        shape = (self.heads, self.kv, self.hd)
        if self.ws is None:
            self.ws = torch.full((max(1, _lib.load().dcd_k_attention_kv4_workspace(len(self.lens), self.T, self.S, *shape)),), 0xFF, dtype=torch.uint8, device="cuda")
        args = (self.q, self.q.stride(0), self.k, self.k.stride(0), self.v, self.v.stride(0), *self.cache, self.S, self.gate, 2 * self.heads * self.hd, self.out,
                self.cu, len(self.lens), self.T, *shape, int(self.causal), self.ws, self.ws.numel(), self.err, st)
        rc = _lib.load().dcd_k_attention_kv4(*[C.c_void_p(a.data_ptr()) if isinstance(a, torch.Tensor) else a for a in args])
        assert rc == 0, rc

    def check(self, rows=None):
        import torch
        torch.cuda.synchronize()
        assert int(self.err.item()) == 0
        ks, vs = values(*self.cache[:2])[:self.S], values(*self.cache[2:])[:self.S]
        at = 0
        for i, n in enumerate(self.lens):
            r = slice(at, at + n)
            at += n
            if n == 0 or (rows is not None and i not in rows):
                continue
            k, v = (torch.cat((a, b[r].double().reshape(n, self.kv, self.hd))) for a, b in ((ks, self.k), (vs, self.v)))
            seen = torch.ones(n, self.S + n, dtype=torch.bool, device="cuda")
            if self.causal:
                seen[:, self.S:] = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
            want, spread = attend(self.q[r], k, v, seen)
            close(self.out[r], want, spread, None if self.gate is None else self.gate[r, :, self.hd:])
        assert (self.out[self.n:] == -7.0).all()  # rows behind the last sequence


SHAPES = [(24, 4, 256), (4, 1, 64), (16, 2, 128), (8, 8, 128), (16, 1, 128), (15, 3, 256), (1, 1, 64), (34, 2, 64)]


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("lens,S,causal,gate", [([1], 0, False, False), ([1], 1, True, True), ([3, 0, 40], 70, False, True), ([5, 130, 1, 64], 129, True, False),
                                                ([127, 128, 129], 128, False, True), ([300], 0, True, True), ([20, 21, 22], 1000, False, False)])
def test_attention_questions(G, heads, kv, hd, lens, S, causal, gate):
    c = Questions(lens, S, heads, kv, hd, causal, gate)
    c.launch(G)
    c.check()


@pytest.mark.parametrize("heads,kv,hd,lens,S,causal", [(24, 4, 256, [16], 4096, False), (24, 4, 256, [16, 5], 16384, False), (16, 2, 128, [1, 2], 9000, True),
                                                       (4, 1, 64, [700, 900], 0, True), (24, 4, 256, [500, 300], 0, True), (16, 1, 128, [33] * 12, 2048, False)])
def test_attention_questions_long(G, heads, kv, hd, lens, S, causal):
    c = Questions(lens, S, heads, kv, hd, causal, True)
    c.launch(G)
    c.check()


@pytest.mark.parametrize("heads,kv,hd", [(24, 4, 256), (16, 2, 128), (4, 1, 64)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_questions_do_not_read_each_other(G, heads, kv, hd, causal):
    """One question's own K/V is NaN and infinity: only its own rows may show it."""
    import torch
    c = Questions([30, 17, 65], 100, heads, kv, hd, causal, False)
    c.k[30:47] = float("nan")
    c.v[30:47] = float("inf")
    c.launch(G)
    torch.cuda.synchronize()
    c.out[30:47] = 0
    c.check(rows=(0, 2))


def test_attention_questions_peaked_and_far_scores(G):
    """Scores of some hundreds, so that nearly all keys weigh nothing and the running maximum grows late."""
    import torch
    for hd, heads, kv in ((256, 24, 4), (128, 16, 2)):
        c = Questions([50, 9], 600, heads, kv, hd, False, False)
        c.q *= 30
        c.launch(G)
        torch.cuda.synchronize()
        ks, vs = values(*c.cache[:2])[:600], values(*c.cache[2:])[:600]
        for r in (slice(0, 50), slice(50, 59)):
            k, v = (torch.cat((a, b[r].double().reshape(-1, kv, hd))) for a, b in ((ks, c.k), (vs, c.v)))
            want, spread = attend(c.q[r], k, v, torch.ones(r.stop - r.start, k.shape[0], dtype=torch.bool, device="cuda"))
            # f32 scores of magnitude up to 2^11: 2^-24 * 256 * 2^11 / 2 in the worst case, a few 2^-24 * 2^11 in the usual: 4e-3 on p.
            # Where the keys that weigh something have a zero in a dimension, the exact value is one of weights below the smallest
            # f32 (2^-126, flushed): 2^-126 * 650 keys * |v| <= 6 is under 1e-34.
            off = (c.out[r].double() - want).abs()
            worst = float((off / (2.0 ** -8 * want.abs() + (2.0 ** -7 + 8e-3) * spread + 1e-34)).max())
            assert torch.isfinite(c.out[r]).all()
            assert worst <= 1, worst


class Decode:
    """One call's operands: stretches in a pool whose other rows hold NaN scales."""

    def __init__(self, lens, L, heads, kv, hd, gate=False, seed=0, max_len=None, behind=2, share=False):
        import torch
        g = gen(seed + sum(lens) + hd + len(lens))
        self.lens, self.heads, self.kv, self.hd = lens, heads, kv, hd
        self.L = [L] * len(lens) if isinstance(L, int) else L
        self.n = sum(self.L)
        self.T = self.n + behind
        self.start, at = [], 1
        for n in lens:
            self.start.append(1 if share else at)
            at += n + 3
        self.pool = at
        self.cache = random_cache(g, at, kv, hd)
        inside = torch.zeros(at, dtype=torch.bool, device="cuda")
        for s, n in zip(self.start, lens):
            inside[s:s + n] = True
        for i in (1, 3):
            self.cache[i][~inside] = 0x7F
        self.max_len = max(lens) if max_len is None else max_len
        self.q = normal(g, self.T, heads * hd + 16, by=1.5)[:, :heads * hd]
        self.gate = normal(g, self.T, heads, 2 * hd) if gate else None
        self.t_start = torch.tensor(self.start, dtype=torch.int64, device="cuda")
        self.t_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.cu = torch.tensor(cu_of(self.L), dtype=torch.int32, device="cuda")
        self.out = torch.full((self.T, heads, hd), -7.0, dtype=torch.bfloat16, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.ws = None

    def launch(self, G, st=None):
        import torch
        from decidra_b200 import _lib
        shape = (self.heads, self.kv, self.hd)
        if self.ws is None:
            self.ws = torch.full((max(1, _lib.load().dcd_k_attention_kv4_decode_workspace(len(self.lens), self.T, self.max_len, *shape)),), 0xFF, dtype=torch.uint8,
                                 device="cuda")
        args = (self.q, self.q.stride(0), *self.cache, self.pool, self.t_start, self.t_len, self.max_len, self.gate, 2 * self.heads * self.hd, self.out, self.cu,
                len(self.lens), self.T, *shape, self.ws, self.ws.numel(), self.err, st)
        rc = _lib.load().dcd_k_attention_kv4_decode(*[C.c_void_p(a.data_ptr()) if isinstance(a, torch.Tensor) else a for a in args])
        assert rc == 0, rc

    def check(self, lens=None, err=0):
        import torch
        torch.cuda.synchronize()
        assert int(self.err.item()) == err
        k, v = values(*self.cache[:2]), values(*self.cache[2:])
        at = 0
        for s, n, L in zip(self.t_start.tolist(), lens or self.lens, self.L):
            seen = torch.arange(n, device="cuda")[None] <= (n - L + torch.arange(L, device="cuda"))[:, None]
            want, spread = attend(self.q[at:at + L].reshape(L, self.heads, self.hd), k[s:s + n], v[s:s + n], seen)
            close(self.out[at:at + L], want, spread, None if self.gate is None else self.gate[at:at + L, :, self.hd:])
            at += L
        assert (self.out[self.n:] == -7.0).all()


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("lens,L", [([1], 1), ([0, 5, 0], 1), ([64, 63, 65, 1, 17], 1), ([300, 2, 129], 3), ([2000], 1), ([15, 16, 31, 33, 128], [2, 1, 5, 0, 9])])
def test_attention_decode(G, heads, kv, hd, lens, L):
    c = Decode(lens, L, heads, kv, hd, gate=len(lens) == 3)
    c.launch(G)
    c.check()


@pytest.mark.parametrize("heads,kv,hd,lens,L", [(24, 4, 256, [16384], 1), (24, 4, 256, [5000, 1, 0, 12345], 1), (16, 2, 128, [30000, 700], 4), (4, 1, 64, [9000] * 3, 2),
                                                (24, 4, 256, [700 + 31 * i for i in range(40)], 1), (16, 1, 128, [4000, 100], 40)])
def test_attention_decode_long(G, heads, kv, hd, lens, L):
    c = Decode(lens, L, heads, kv, hd)
    c.launch(G)
    c.check()


def test_attention_decode_shared_stretch_and_loose_bound(G):
    c = Decode([500, 400, 500, 3], 2, 16, 2, 128, share=True, max_len=5000)
    c.launch(G)
    c.check()


def test_attention_decode_bad_stretches_give_zero_and_set_the_error_word(G):
    import torch
    c = Decode([50, 60, 70, 80, 90], 1, 24, 4, 256)
    c.t_start[1] = -1
    c.t_start[2] = c.pool - 5
    c.t_start[3] = 2 ** 62
    c.max_len = 89
    c.launch(G)
    torch.cuda.synchronize()
    assert int(c.err.item()) == 7
    assert (c.out[1:5] == 0).all()
    want, spread = attend(c.q[:1].reshape(1, 24, 256), values(*c.cache[:2])[1:51], values(*c.cache[2:])[1:51], torch.ones(1, 50, dtype=torch.bool, device="cuda"))
    close(c.out[:1], want, spread)
    assert (c.out[5:] == -7.0).all()


def test_attention_offsets_beyond_32_bits(G):
    """A pool whose code arrays are over 4 GiB each: the rows at its end."""
    import torch
    rows, kv, hd = 9_000_000, 4, 256
    free, _ = torch.cuda.mem_get_info()
    if free < 30 << 30:
        pytest.skip("needs 12 GB of device memory")
    cache = [torch.zeros((rows, kv, hd // n), dtype=torch.uint8, device="cuda") for n in (2, 16, 2, 16)]
    n = 300
    small = random_cache(gen(3), n, kv, hd)
    g = gen(4)
    k, v = normal(g, 1, kv * hd), normal(g, 1, kv * hd)
    err = G.devi([0])
    for c, s in zip(cache, small):
        c[rows - n:] = s
    G.call("dcd_k_kv4_write", k, kv * hd, v, kv * hd, torch.tensor([rows - 1], device="cuda"), *cache, rows, 1, kv, hd, 1, err, None)
    for c, s in zip(cache, small):
        s[n - 1] = c[rows - 1]
    assert torch.equal(values(*small[:2])[n - 1].reshape(1, -1), encoded(k))
    d = Decode([n], 1, 24, kv, hd)
    d.cache, d.pool = cache, rows
    d.t_start[0] = rows - n
    d.launch(G)
    torch.cuda.synchronize()
    assert int(d.err.item()) == 0
    want, spread = attend(d.q[:1].reshape(1, 24, hd), values(*small[:2]), values(*small[2:]), torch.ones(1, n, dtype=torch.bool, device="cuda"))
    close(d.out[:1], want, spread)


@pytest.mark.parametrize("lens", [[(7 * i) % 45 for i in range(40)], [(5 * i) % 23 for i in range(131)], [1] * 33])
@pytest.mark.parametrize("heads,kv,hd,S", [(16, 2, 128, 0), (24, 4, 256, 140), (8, 8, 64, 3)])
def test_attention_causal_prompts_by_the_dozen(G, heads, kv, hd, S, lens):
    """More prompts than a warp has lanes, and more than its lanes hold: the order of the work changes, not the result."""
    c = Questions(lens, S, heads, kv, hd, True, False)
    c.launch(G)
    c.check()


@pytest.mark.parametrize("causal,lens", [(True, [1 + (37 * i) % 200 for i in range(100)]), (False, [1 + i % 3 for i in range(200)])])
def test_attention_more_items_than_one_wave_lists(G, causal, lens):
    """64 K/V heads, a query head each: about ten thousand work items."""
    c = Questions(lens, 0, 64, 64, 64, causal, False)
    c.launch(G)
    c.check()


BAD_OFFSETS = [([0, 5, 3, 12], [0]), ([-1, 4, 9, 12], [1, 2]), ([0, 4, 99, 12], [0]), ([0, 4, 12, -2 ** 31], [0, 1]), ([2 ** 31 - 1, 4, 9, 12], [1, 2])]


@pytest.mark.parametrize("cu,good", BAD_OFFSETS)
@pytest.mark.parametrize("causal,S", [(False, 300), (True, 0), (False, 5000)])
def test_attention_questions_with_bad_offsets(G, cu, good, causal, S):
    """A sequence whose offsets fall or leave the batch is left out and reported; the sound ones beside it are computed, and rows that
    belong to none stay as they were. ([0, 5, 3, 12]: rows 3 and 4 would be two sequences' and are not looked at.)"""
    import torch
    c = Questions([5, 4, 3], S, 16, 2, 128, causal, False, behind=0)
    c.cu.copy_(torch.tensor(cu, dtype=torch.int32))
    c.launch(G)
    torch.cuda.synchronize()
    assert int(c.err.item()) == 8
    ks, vs = values(*c.cache[:2])[:S], values(*c.cache[2:])[:S]
    taken = set()
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        if not 0 <= a <= b <= c.T:
            continue
        taken |= set(range(a, b))
        if i not in good:
            continue
        stop = 3 if cu[:3] == [0, 5, 3] else b  # its later rows are another sequence's too
        n = b - a
        k, v = (torch.cat((x, y[a:b].double().reshape(n, 2, 128))) for x, y in ((ks, c.k), (vs, c.v)))
        seen = torch.ones(n, S + n, dtype=torch.bool, device="cuda")
        if causal:
            seen[:, S:] = seen[:, S:].tril()
        want, spread = attend(c.q[a:b], k, v, seen)
        close(c.out[a:stop], want[:stop - a], spread[:stop - a])
    rest = [t for t in range(c.T) if t not in taken]
    assert (c.out[rest] == -7.0).all()


@pytest.mark.parametrize("causal,S", [(False, 300), (True, 0), (False, 5000)])
def test_attention_questions_with_offsets_that_cover_the_batch_many_times(G, causal, S):
    """Falling offsets whose sound pairs hold far more tokens than the batch: reported, nothing computed, nothing written."""
    import torch
    c = Questions([1] * 400, S, 16, 2, 128, causal, False, behind=0)
    c.cu.copy_(torch.tensor([400 * (i % 2) for i in range(401)], dtype=torch.int32))
    c.launch(G)
    torch.cuda.synchronize()
    assert int(c.err.item()) == 8
    assert (c.out == -7.0).all()


@pytest.mark.parametrize("cu,good", BAD_OFFSETS)
def test_attention_decode_with_bad_offsets(G, cu, good):
    import torch
    c = Decode([50, 3000, 70], [5, 4, 3], 16, 2, 128, behind=0)
    c.cu.copy_(torch.tensor(cu, dtype=torch.int32))
    c.launch(G)
    torch.cuda.synchronize()
    assert int(c.err.item()) == 8
    k, v = values(*c.cache[:2]), values(*c.cache[2:])
    taken = set()
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        if not 0 <= a <= b <= c.T:
            continue
        taken |= set(range(a, b))
        if i not in good or cu[:3] == [0, 5, 3]:
            continue
        s, n, L = c.start[i], c.lens[i], b - a
        seen = torch.arange(n, device="cuda")[None] <= (n - L + torch.arange(L, device="cuda"))[:, None]
        close(c.out[a:b], *attend(c.q[a:b].reshape(L, 16, 128), k[s:s + n], v[s:s + n], seen))
    rest = [t for t in range(c.T) if t not in taken]
    assert (c.out[rest] == -7.0).all()


def test_attention_decode_many_sequences(G):
    """More sequences than a CTA has threads, most of them short, under a bound far above them."""
    c = Decode([(13 * i) % 71 for i in range(600)], 1, 4, 1, 64, max_len=1 << 14)
    c.launch(G)
    c.check()


def test_attention_same_bits_every_run(G):
    import torch
    for c in (Questions([40, 90, 1], 3000, 24, 4, 256, False, True), Questions([200, 31], 0, 16, 2, 128, True, False), Decode([5000, 77, 1234], 2, 24, 4, 256)):
        c.launch(G)
        torch.cuda.synchronize()
        first = c.out.clone()
        for i in range(6):
            c.ws.fill_((0x7F, 0xFF, 0x00)[i % 3])
            c.out.fill_(-7.0)
            c.launch(G)
            torch.cuda.synchronize()
            assert torch.equal(first, c.out)


def test_attention_in_graphs_and_on_streams(G):
    """Captured once and replayed with other lengths, while another call runs on a stream of its own."""
    import torch
    a = Decode([900, 30, 2000], 1, 24, 4, 256, max_len=2000)
    b = Questions([33, 20], 700, 24, 4, 256, False, True)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for c, s in ((a, s1), (b, s2)):  # the workspace and the first launch come before the capture
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            c.launch(G, C.c_void_p(s.cuda_stream))
    torch.cuda.synchronize()
    a.check()
    b.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s1):
        a.launch(G, C.c_void_p(torch.cuda.current_stream().cuda_stream))
    for lens in ([900, 30, 2000], [1, 0, 1999], [899, 29, 64]):
        a.t_len.copy_(torch.tensor(lens, dtype=torch.int32))
        a.out.fill_(-7.0)
        b.out.fill_(-7.0)
        torch.cuda.synchronize()
        graph.replay()
        b.launch(G, C.c_void_p(s2.cuda_stream))
        torch.cuda.synchronize()
        a.check(lens)
        b.check()


def test_attention_questions_captured_and_replayed(G):
    """The state's decoding and the attention that starts under it, in one graph: replayed with another state and other offsets."""
    import torch
    for c in (Questions([33, 20, 0], 700, 24, 4, 256, False, True), Questions([5, 2, 1], 5000, 16, 2, 128, True, False)):
        c.launch(G)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.launch(G, C.c_void_p(torch.cuda.current_stream().cuda_stream))
        for seed, lens in ((1, c.lens), (2, [c.lens[0] - 3, 3, c.lens[1] + c.lens[2]])):
            for old, new in zip(c.cache, random_cache(gen(seed), c.S + 2, c.kv, c.hd)):
                old[:c.S] = new[:c.S]
            c.lens = lens
            c.cu.copy_(torch.tensor(cu_of(lens), dtype=torch.int32))
            c.out.fill_(-7.0)
            graph.replay()
            c.check()


def test_layer_step_with_all_of_them(G):
    """One low-precision attention layer as a server runs it: residual + norm to e4m3, the FP8 product to q/k/v, the state's K/V into
    the cache, questions over it; then new tokens appended and attended to. Every step against 64 bits on what the step was given."""
    import torch
    g = gen(11)
    H, heads, kv, hd, S, lens = 512, 24, 4, 256, 200, [30, 41]
    N = (heads + 2 * kv) * hd
    T = S + sum(lens)
    x, mix, w = normal(g, T, H, by=2.0), normal(g, T, H), normal(g, H, by=0.1)
    wt = normal(g, N, H, by=0.05)
    wq, wsc = torch.empty((N, H), dtype=torch.uint8, device="cuda"), torch.empty(N, device="cuda")
    G.call("dcd_k_quant_fp8_rows", wt, C.c_size_t(H), wq, wsc, N, H, C.c_float(1.0), 1, None)
    q8, sc, res = norm_call(G, x, mix, w, H, round_t=1)
    norm = (res.double() / torch.sqrt(res.double().square().mean(1, keepdim=True) + 1e-6) * (1 + w.double()))
    qkv, err = torch.empty((T, N), dtype=torch.bfloat16, device="cuda"), G.devi([0])
    G.call("dcd_k_gemm_fp8_tc", q8, wq, qkv, T, N, H, N, 0, sc, wsc, G.sm_count(), err, None)
    assert int(err.item()) == 0
    want = norm @ (wq.view(torch.float8_e4m3fn).double() * wsc.double()[:, None]).T
    # e4m3 rounds each of H inputs by up to 2^-4 of it (2^-5 rms at random signs): 6 standard deviations of the sum
    spread = torch.sqrt(norm.square() @ (wt.double().T.square()))
    assert ((qkv.double() - want).abs() <= 6 * 2.0 ** -5 * spread + 2.0 ** -7 * want.abs() + 1e-3).all()
    q, k, v = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kv) * hd], qkv[:, (heads + kv) * hd:]
    pool = S + 50
    cache = new_cache(pool, kv, hd)
    G.call("dcd_k_kv4_write", k, N, v, N, None, *cache, pool, S, kv, hd, 1, err, None)
    assert torch.equal(values(*cache[:2])[:S].reshape(S, -1), encoded(k[:S]))
    c = Questions(lens, S, heads, kv, hd, False, False, behind=0)
    c.q, c.k, c.v, c.cache = q[S:], k[S:], v[S:], cache
    c.launch(G)
    torch.cuda.synchronize()
    ks, vs = values(*cache[:2])[:S], values(*cache[2:])[:S]
    for r in (slice(S, S + 30), slice(S + 30, T)):
        n = r.stop - r.start
        kk, vv = (torch.cat((a, b[r].double().reshape(n, kv, hd))) for a, b in ((ks, k), (vs, v)))
        close(c.out[r.start - S:r.stop - S], *attend(q[r].reshape(n, heads, hd), kk, vv, torch.ones(n, S + n, dtype=torch.bool, device="cuda")))
    # the state is continued by three tokens: written behind it, then attended to with it
    G.call("dcd_k_kv4_write", k[S:], N, v[S:], N, torch.arange(S, S + 3, device="cuda"), *cache, pool, 3, kv, hd, 1, err, None)
    d = Decode([S + 3], 3, heads, kv, hd, behind=0)
    d.q, d.cache, d.pool = q[S:S + 3], cache, pool
    d.t_start[0] = 0
    d.launch(G)
    torch.cuda.synchronize()
    assert int(d.err.item()) == 0 and int(err.item()) == 0
    seen = torch.arange(S + 3, device="cuda")[None] <= torch.arange(S, S + 3, device="cuda")[:, None]
    close(d.out, *attend(q[S:S + 3].reshape(3, heads, hd), values(*cache[:2])[:S + 3], values(*cache[2:])[:S + 3], seen))
