"""The low-precision attention layer's kernels where they can go wrong unnoticed: work items of one key tile, values that are not finite
in calls whose keys are split, loose bounds, offsets that fall, operands off their alignment, and every key counted once."""
import ctypes as C
import math

import pytest

from test_gpu_kv4 import Decode, Questions, attend, cu_of, gen, norm_call, norm_check, normal, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def G(dcd):
    import torch
    assert torch.cuda.is_available()
    import gpu_util
    return gpu_util


# ---------------------------------------------------------------------------------------------
# items of one key tile
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("causal", [False, True])
def test_items_of_one_key_tile_behind_each_other(G, hd, causal):
    """Twenty items a CTA, nearly all of a single key tile, whose sums differ by up to a hundred times: each row is divided by its own
    sum, whichever group of warps has the tile and however far the other one is behind."""
    import torch
    lens = [(1 + (37 * i) % 120, 130 + i)[i % 29 == 28] for i in range(200)]
    c = Questions(lens, 0, 16, 16, hd, causal, False)
    c.launch(G)
    c.check(rows=range(0, 200, 3))
    first = c.out.clone()
    for _ in range(3):
        c.out.fill_(-7.0)
        c.launch(G)
        torch.cuda.synchronize()
        assert torch.equal(first, c.out)


# ---------------------------------------------------------------------------------------------
# values that are not finite
# ---------------------------------------------------------------------------------------------
NAN, INF = float("nan"), float("inf")


def near(got, want, spread):
    """The bound of test_gpu_kv4.close, where the value is finite."""
    off = (got.double() - want).abs()
    assert (off <= 2.0 ** -8 * want.abs() + (2.0 ** -7 + 1e-3) * spread + 1e-30).all()


@pytest.mark.parametrize("heads,kv,hd", [(24, 4, 256), (16, 2, 128), (4, 1, 64)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("where", ["query", "query inf", "own key", "every own key", "state key", "own value", "state value"])
def test_questions_show_a_nan_whether_their_keys_are_split_or_not(G, heads, kv, hd, causal, where):
    """One question over a long state has its keys split into parts, the same one among a hundred others has not: a NaN shows in the rows
    that see it, in both, and nowhere else."""
    import torch
    n, S, kh, rep = 16, 4000, kv - 1, heads // kv
    for others in (0, 160):
        c = Questions([n] + [20] * others, S, heads, kv, hd, causal, False)
        ks, vs = values(*c.cache[:2])[:S], values(*c.cache[2:])[:S]
        seen = torch.ones(n, S + n, dtype=torch.bool, device="cuda")
        if causal:
            seen[:, S:] = seen[:, S:].tril()
        want, spread = attend(c.q[:n], torch.cat((ks, c.k[:n].double().reshape(n, kv, hd))), torch.cat((vs, c.v[:n].double().reshape(n, kv, hd))), seen)
        bad = torch.zeros(n, heads, hd, dtype=torch.bool, device="cuda")
        group = slice(kh * rep, (kh + 1) * rep)
        if where.startswith("query"):
            c.q[5, 1, 7] = INF if where.endswith("inf") else NAN  # infinite scores of either sign: NaN as well
            bad[5, 1] = True
        elif where == "own key":
            c.k[6, kh * hd + 3] = NAN
            bad[6 if causal else 0:, group] = True
        elif where == "every own key":
            c.k[:n, kh * hd + 3] = NAN
            bad[:, group] = True
        elif where == "state key":
            c.cache[1][1234, kh, 0] = 0x7F
            bad[:, group] = True
        elif where == "own value":
            c.v[0, kh * hd + 3] = NAN
            bad[:, group, 3] = True
        else:
            c.cache[3][1234, kh, 1] = 0x7F
            bad[:, group, 16:32] = True
        c.launch(G)
        torch.cuda.synchronize()
        assert int(c.err.item()) == 0
        got = c.out[:n]
        assert torch.equal(torch.isnan(got), bad)
        near(got[~bad], want[~bad], spread[~bad])


@pytest.mark.parametrize("heads,kv,hd", [(24, 4, 256), (16, 2, 128), (4, 1, 64), (16, 4, 128)])
@pytest.mark.parametrize("where", ["query", "query inf", "key", "every key", "value"])
def test_new_tokens_show_a_nan_whether_their_keys_are_split_or_not(G, heads, kv, hd, where):
    """The same in the form for new tokens: three drafted tokens over a stretch that one warp takes, over one of many parts, and beside one
    that is too short for the first two (they see no row and give 0, whatever they ask)."""
    import torch
    L, kh, rep = 3, kv - 1, heads // kv
    for n in (20, 6000):
        c = Decode([n, 1], L, heads, kv, hd)
        s, s1 = c.start
        k, v = values(*c.cache[:2]), values(*c.cache[2:])
        seen = torch.arange(n, device="cuda")[None] <= (n - L + torch.arange(L, device="cuda"))[:, None]
        want, spread = attend(c.q[:L].reshape(L, heads, hd), k[s:s + n], v[s:s + n], seen)
        bad = torch.zeros(L, heads, hd, dtype=torch.bool, device="cuda")
        group = slice(kh * rep, (kh + 1) * rep)
        if where.startswith("query"):
            c.q[1, hd + 7] = INF if where.endswith("inf") else NAN
            bad[1, 1] = True
            c.q[L:L + 2] = NAN
        elif where == "key":
            c.cache[1][s + n - 2, kh, 0] = 0x7F  # the first token does not see it
            bad[1:, group] = True
        elif where == "every key":
            c.cache[1][s:s + n, kh, 0] = 0x7F
            bad[:, group] = True
        else:
            c.cache[3][s + 7, kh, 1] = 0x7F
            bad[:, group, 16:32] = True
        c.launch(G)
        torch.cuda.synchronize()
        assert int(c.err.item()) == 0
        got = c.out[:L]
        assert torch.equal(torch.isnan(got), bad)
        near(got[~bad], want[~bad], spread[~bad])
        assert (c.out[L:L + 2] == 0).all() and (c.out[2 * L:] == -7.0).all()


# ---------------------------------------------------------------------------------------------
# the bound on the lengths
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv,hd", [(24, 4, 256), (16, 2, 128), (4, 1, 64)])
def test_a_loose_bound_on_the_lengths_costs_no_time(G, heads, kv, hd):
    """64 sequences of about a thousand rows, called with their longest length and with a context limit of 131072."""
    import torch
    took = []
    for bound in (None, 131072):
        c = Decode([900 + 3 * i for i in range(64)], 1, heads, kv, hd, max_len=bound)
        c.launch(G)
        c.check()
        times = []
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                c.launch(G)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        took.append(sorted(times)[5])
    assert took[1] < 2 * took[0], took


@pytest.mark.parametrize("heads,kv,hd", [(24, 4, 256), (16, 2, 128), (4, 1, 64), (15, 3, 256)])
@pytest.mark.parametrize("bound", [None, 1 << 30])
def test_new_tokens_of_very_different_lengths(G, heads, kv, hd, bound):
    """One long stretch among many short ones, whose keys then go to hundreds of parts, and sequences with more tokens than a round."""
    c = Decode([5 + i % 90 for i in range(70)] + [40000] + [3, 0, 700], [1] * 70 + [2, 40, 1, 17], heads, kv, hd, gate=True, max_len=bound)
    c.launch(G)
    c.check()


# ---------------------------------------------------------------------------------------------
# offsets
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cu", [[0, 99, 3, 12], [5, 2 ** 31 - 1, 0, 12], [-7, 9, 2, 12], [0, 4, 99, 4, 12]])
@pytest.mark.parametrize("heads,kv,hd", [(16, 2, 128), (24, 4, 256)])
def test_new_tokens_of_a_sound_sequence_behind_offsets_that_fall(G, cu, heads, kv, hd):
    """Its keys are split into parts, which have to be added up whatever the offsets in front of it are."""
    import torch
    n = len(cu) - 1
    c = Decode([5000, 60, 3000, 7000][:n], [4] * n, heads, kv, hd, behind=0)
    c.T = 12
    c.cu.copy_(torch.tensor(cu, dtype=torch.int32))
    c.launch(G)
    torch.cuda.synchronize()
    assert int(c.err.item()) == 8
    k, v = values(*c.cache[:2]), values(*c.cache[2:])
    taken = set()
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        if 0 <= a <= b <= c.T:
            taken |= set(range(a, b))
            s, m, L = c.start[i], c.lens[i], b - a
            seen = torch.arange(m, device="cuda")[None] <= (m - L + torch.arange(L, device="cuda"))[:, None]
            near(c.out[a:b], *attend(c.q[a:b].reshape(L, heads, hd), k[s:s + m], v[s:s + m], seen))
    assert (c.out[[t for t in range(12) if t not in taken]] == -7.0).all()


def test_new_tokens_rows_behind_the_last_sequence_cost_little(G):
    """A call at a server's capacity: 4096 sequences, and room for twice as many tokens as they have."""
    import torch
    took = []
    for behind in (0, 4096):
        c = Decode([5] * 4096, 1, 24, 4, 256, behind=behind)
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            c.launch(G)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        took.append(sorted(times)[2])
        assert (c.out[c.n:] == -7.0).all()
    assert took[1] < 1.5 * took[0], took


# ---------------------------------------------------------------------------------------------
# the norm's rounded form
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,cols", [(200, 8), (20000, 1024), (8000, 5120), (200, 8192), (200, 8200)])
@pytest.mark.parametrize("off", ["stride", "x", "w", "mix", "residual", "out", "all"])
def test_rounded_norm_has_the_bits_of_the_two_calls_off_16_bytes_too(G, dtype, rows, cols, off):
    """Rows inside a wider matrix of an odd stride, and operands an element (the codes: a byte) off their alignment: the sum of squares keeps
    the order of the two calls on aligned copies. (Another order moves 1 / sqrt by a unit of its last place, which shows in a few of ten
    million codes.)"""
    import torch
    g = gen(cols + rows)
    x, mix, w = normal(g, rows, cols, dtype=dtype, by=2.0), normal(g, rows, cols, dtype=dtype), normal(g, cols, dtype=dtype, by=0.1)

    def place(a, name, stride=None):  # a copy that lies an element further on, or with another stride
        shift = 1 if off in (name, "all") else 0
        stride = stride or cols
        whole = torch.zeros(rows * stride + 16, dtype=a.dtype, device="cuda")
        return torch.as_strided(whole, a.shape, (stride, 1) if a.dim() == 2 else (1,), shift).copy_(a)

    wide = cols + 3 if off in ("stride", "all") else cols
    xs, ms, ws = place(x, "x", wide), place(mix, "mix", wide), place(w, "w")
    for add in (False, True):
        y, r = torch.empty_like(x), torch.empty_like(x)
        if add:
            G.call("dcd_k_add_rmsnorm", x, mix, w, r, y, rows, cols, C.c_float(1e-6), dtype, None)
        else:
            G.call("dcd_k_rmsnorm", x, w, y, rows, cols, C.c_float(1e-6), 1, dtype, None)
        q, sc = torch.empty((rows, cols), dtype=torch.uint8, device="cuda"), torch.empty(rows, device="cuda")
        G.call("dcd_k_quant_fp8_rows", y, C.c_size_t(cols), q, sc, rows, cols, C.c_float(1.0), dtype, None)
        q2, sc2 = place(torch.zeros_like(q), "out"), torch.empty_like(sc)
        if add:
            r2 = place(torch.zeros_like(r), "residual")
            G.call("dcd_k_add_rmsnorm_fp8", xs, xs.stride(0), ms, ms.stride(0), ws, r2, q2, sc2, rows, cols, 1e-6, 1, 1.0, 1, dtype, None)
            assert torch.equal(r, r2)
        else:
            G.call("dcd_k_rmsnorm_fp8", xs, xs.stride(0), ws, q2, sc2, rows, cols, 1e-6, 1, 1.0, 1, dtype, None)
        assert torch.equal(sc, sc2) and torch.equal(q, q2)


@pytest.mark.parametrize("add", [False, True])
def test_rounded_norm_of_narrow_rows_is_not_slower_than_the_two_calls(G, add):
    import torch
    from decidra_b200 import _lib
    lib, rows, cols = _lib.load(), 20000, 256
    g = gen(8)
    x, mix, w = normal(g, rows, cols), normal(g, rows, cols), normal(g, cols, by=0.1)
    y, r, q, sc = torch.empty_like(x), torch.empty_like(x), torch.empty((rows, cols), dtype=torch.uint8, device="cuda"), torch.empty(rows, device="cuda")
    px, pm, pw, py, pr, pq, ps = (C.c_void_p(a.data_ptr()) for a in (x, mix, w, y, r, q, sc))

    def two():
        if add:
            assert lib.dcd_k_add_rmsnorm(px, pm, pw, pr, py, rows, cols, 1e-6, 1, None) == 0
        else:
            assert lib.dcd_k_rmsnorm(px, pw, py, rows, cols, 1e-6, 1, 1, None) == 0
        assert lib.dcd_k_quant_fp8_rows(py, cols, pq, ps, rows, cols, 1.0, 1, None) == 0

    def one():
        if add:
            assert lib.dcd_k_add_rmsnorm_fp8(px, cols, pm, cols, pw, pr, pq, ps, rows, cols, 1e-6, 1, 1.0, 1, 1, None) == 0
        else:
            assert lib.dcd_k_rmsnorm_fp8(px, cols, pw, pq, ps, rows, cols, 1e-6, 1, 1.0, 1, 1, None) == 0

    took = []
    for call in (two, one):
        times = []
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                call()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        took.append(sorted(times)[5])
    assert took[1] < took[0], took


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,cols", [(147, 5120), (149, 5120), (9500, 64), (20000, 256), (2000, 1024), (900, 4096)])
def test_norm_of_many_rows(G, dtype, rows, cols):
    """Fewer rows than a wave has CTAs, a few more, and many: every CTA takes its rows in turn."""
    g = gen(rows)
    x, mix, w = normal(g, rows, cols, dtype=dtype, by=3.0), normal(g, rows, cols, dtype=dtype), normal(g, cols, dtype=dtype, by=0.1)
    norm_check(x, None, w, 1, 1.0, *norm_call(G, x, None, w, cols))
    norm_check(x, mix, w, 1, 1.0, *norm_call(G, x, mix, w, cols))


# ---------------------------------------------------------------------------------------------
# the gate
# ---------------------------------------------------------------------------------------------
def test_questions_have_one_gate_whether_their_keys_are_split_or_not(G):
    """Scores of 0 over 4096 keys with V = 1 make 1 exactly, in one part or many: what is left is the gate's value, for every bf16 gate of
    a magnitude below 128."""
    import torch
    n, S, heads, kv, hd = 16, 4080, 24, 4, 256
    bits = torch.arange(0x4300, dtype=torch.int32, device="cuda")
    gates = torch.cat((bits, bits + 0x8000)).to(torch.int16).view(torch.bfloat16)
    outs = []
    for others in (0, 160):
        c = Questions([n] * (1 + others), S, heads, kv, hd, False, True)
        c.q.zero_()
        c.k.zero_()
        c.v.fill_(1.0)
        c.cache[2].fill_(0x22)
        c.cache[3].fill_(0x38)
        c.gate[:n, :, hd:] = gates.repeat(3)[:n * heads * hd].reshape(n, heads, hd)
        c.launch(G)
        torch.cuda.synchronize()
        assert int(c.err.item()) == 0
        outs.append(c.out[:n].clone())
    want = torch.sigmoid(gates.double()).repeat(3)[:n * heads * hd].reshape(n, heads, hd)
    assert ((outs[0].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -21) * want + 2.0 ** -126).all()
    assert torch.equal(outs[0], outs[1])


# ---------------------------------------------------------------------------------------------
# every key once
# ---------------------------------------------------------------------------------------------
ONE = 0x38  # 1.0 in e4m3


def dimension_of(j, hd, fine):
    """The dimension in which key j has its only value: neighbouring keys in neighbouring ones, or sixteen keys in one."""
    return (j if fine else j // 16) % hd


def counting(codes, hd, j, fine):
    """The rows of codes for keys j: 6 in one dimension, 0 elsewhere."""
    import torch
    d = dimension_of(j, hd, fine)
    codes.zero_()
    codes[torch.arange(len(j), device="cuda"), :, d // 2] = torch.where(d % 2 == 0, 7, 0x70).to(torch.uint8)[:, None].expand(-1, codes.shape[1])


def counted(got, sees, hd, fine):
    """With all scores 0 a token that sees n keys gives 6 / n for each one that has its value in a dimension: exact but for the division's and
    the output's rounding. In the fine form a key that is missing, or there twice, is one of at most 128; in the other sixteen keys are."""
    import torch
    for i, n in enumerate(sees):
        want = torch.bincount(dimension_of(torch.arange(n, device="cuda"), hd, fine), minlength=hd).double() * 6 / max(n, 1)
        assert ((got[i].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -21) * want).all(), (i, n)


COUNTS = [(24, 4, 256), (16, 2, 128), (4, 1, 64), (15, 3, 256), (8, 8, 64)]


@pytest.mark.parametrize("heads,kv,hd", COUNTS)
@pytest.mark.parametrize("lens,L,fine", [([16384], 1, True), ([30000, 700, 1, 0, 33], 4, False), ([100 + 37 * i for i in range(40)], 1, True), ([12345, 64, 31, 5000], 2, True),
                                         ([100000], 1, False)])
def test_new_tokens_count_every_key_once(G, heads, kv, hd, lens, L, fine):
    import torch
    fine = fine and max(lens) <= 128 * hd
    c = Decode(lens, L, heads, kv, hd)
    c.q.zero_()
    for s, n in zip(c.start, lens):
        counting(c.cache[2][s:s + n], hd, torch.arange(n, device="cuda"), fine)
        c.cache[3][s:s + n] = ONE
    c.launch(G)
    torch.cuda.synchronize()
    assert int(c.err.item()) == 0
    counted(c.out[:c.n], [max(0, n - L + 1 + i) for n in lens for i in range(L)], hd, fine)


@pytest.mark.parametrize("heads,kv,hd", COUNTS)
@pytest.mark.parametrize("lens,S,causal", [([16], 4096, False), ([16, 5], 16000, True), ([1], 1025, False), ([20] * 60, 2049, False), ([700, 900], 0, True), ([500, 127, 129, 1], 300, True),
                                           ([1500], 0, False)])
def test_questions_count_every_key_once(G, heads, kv, hd, lens, S, causal):
    import torch
    fine = S <= 100 * hd
    c = Questions(lens, S, heads, kv, hd, causal, False)
    c.q.zero_()
    counting(c.cache[2][:S], hd, torch.arange(S, device="cuda"), fine)
    c.cache[3][:S] = ONE
    at, sees = 0, []
    for n in lens:
        d = dimension_of(torch.arange(S, S + n, device="cuda"), hd, fine)
        own = torch.zeros(n, kv, hd, device="cuda", dtype=torch.bfloat16)
        own[torch.arange(n, device="cuda"), :, d] = 6.0
        c.v[at:at + n] = own.reshape(n, kv * hd)
        sees += [S + (i + 1 if causal else n) for i in range(n)]
        at += n
    c.launch(G)
    torch.cuda.synchronize()
    assert int(c.err.item()) == 0
    counted(c.out[:c.n], sees, hd, fine)


@pytest.mark.parametrize("heads,kv,hd", [(24, 4, 256), (16, 2, 128), (4, 1, 64)])
@pytest.mark.parametrize("lens,L", [([2000] * 64, 1), ([40000], 1), ([3000] * 20, 4), ([33] * 40, 2)])
def test_new_tokens_find_one_key_wherever_it_is(G, heads, kv, hd, lens, L):
    """A key whose score is hundreds above all others, at blocks' and parts' borders and in the last rows: its value comes back exactly."""
    import torch
    c = Decode(lens, L, heads, kv, hd)
    c.q.fill_(1.0)
    n, v = lens[0], values(*c.cache[2:])
    spots = [0, 31, 32, n - L, n // 2, n - 33, n - 32] + [(2 * i + 1) * n // 120 for i in range(60)] + [32 * i % n for i in range(5, 400, 13)] + [32 * i % n + 31 for i in range(7, 400, 31)]
    spots = [p for p in spots if 0 <= p <= n - L]
    for first in range(0, len(spots), len(lens)) if len(lens) > 1 else range(0, len(spots), 6):
        planted = [(spots + spots)[(first + b) % len(spots)] for b in range(len(lens))]
        c.cache[0].zero_()
        for s, p in zip(c.start, planted):
            c.cache[0][s + p] = 0x77
            c.cache[1][s:s + n] = ONE
            c.cache[1][s + p] = 0x50  # 8: the key is 48 in every dimension
        c.launch(G)
        torch.cuda.synchronize()
        assert int(c.err.item()) == 0
        want = torch.stack([v[s + p] for s, p in zip(c.start, planted) for _ in range(L)]).repeat_interleave(heads // kv, 1)
        assert torch.equal(c.out[:c.n].double(), want), planted


@pytest.mark.parametrize("heads,kv,hd", [(24, 4, 256), (16, 2, 128), (4, 1, 64)])
@pytest.mark.parametrize("lens,S", [([16], 4096), ([5, 9], 16001), ([20] * 64, 2048), ([300, 200], 100)])
@pytest.mark.parametrize("causal", [False, True])
def test_questions_find_one_key_wherever_it_is(G, heads, kv, hd, lens, S, causal):
    import torch
    c = Questions(lens, S, heads, kv, hd, causal, False)
    c.q.fill_(1.0)
    vs = values(*c.cache[2:])[:S]
    c.k.zero_()
    for p in [0, 15, 16, 127, 128, 129, S - 1, S - 128, S // 2, S // 3] + [S * i // 13 // 128 * 128 + (i % 3 - 1) * 127 for i in range(1, 13)]:
        p = min(max(p, 0), S - 1)
        c.cache[0][:S].zero_()
        c.cache[1][:S] = ONE
        c.cache[0][p], c.cache[1][p] = 0x77, 0x50
        c.launch(G)
        torch.cuda.synchronize()
        assert int(c.err.item()) == 0
        assert torch.equal(c.out[:c.n].double(), vs[p].repeat_interleave(heads // kv, 0).expand(c.n, heads, hd)), p
    # one of the question's own: its last key, which under causal only the last token sees
    c.cache[0][:S].zero_()
    ends = torch.tensor(cu_of(lens)[1:], device="cuda") - 1
    c.k[ends] = 48.0
    c.launch(G)
    torch.cuda.synchronize()
    for a, b in zip(cu_of(lens), cu_of(lens)[1:]):
        rows = slice(b - 1, b) if causal else slice(a, b)
        assert torch.equal(c.out[rows], c.v[b - 1].reshape(kv, hd).repeat_interleave(heads // kv, 0).expand(rows.stop - rows.start, heads, hd))


def rounded_within(got, q, k, v, seen, p_step):
    """A bound on each row's error as a whole. The output's rounding is at most 2^-8 of it; the weights' roundings, at most p_step of each, are
    independent of one another and of the values, so that in the mean over the dimensions they add up as squares: p_step * sqrt(sum p^2 v^2).
    Half as much again covers the mean's own scatter over 64 dimensions and more. A block of 32 keys of some thousand, left out or taken
    twice, is more than twice that, where it is a small part of the bound on a single value."""
    import torch
    rep = q.shape[1] // k.shape[1]
    k, v = (a.double().repeat_interleave(rep, 1) for a in (k, v))
    s = torch.einsum("ihd,jhd->hij", q.double(), k) / math.sqrt(q.shape[2])
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    want = torch.einsum("hij,jhd->ihd", p, v)
    noise = torch.einsum("hij,jhd->ihd", p.square(), v.square()).mean(-1).sqrt()
    off = (got.double() - want).square().mean(-1).sqrt()
    bound = 2.0 ** -8 * want.square().mean(-1).sqrt() + 1.5 * p_step * noise
    assert (off <= bound).all(), float((off / bound).max())
    # ... and the bound sees a block: the same rows without the last 32 keys that all of them see
    m = int(seen.all(0).nonzero().max()) + 1
    if m > 1000:
        less = seen.clone()
        less[:, m - 32:m] = False
        p = torch.softmax(s.masked_fill(~less, -math.inf), -1)
        short = (torch.einsum("hij,jhd->ihd", p, v) - want).square().mean(-1).sqrt()
        assert (short > bound).double().mean() > 0.9


@pytest.mark.parametrize("heads,kv,hd,lens,L", [(24, 4, 256, [16384], 1), (24, 4, 256, [5000, 1, 12345], 1), (16, 2, 128, [30000, 700], 4), (4, 1, 64, [9000] * 3, 2), (16, 1, 128, [4000, 100], 40)])
def test_new_tokens_whole_rows(G, heads, kv, hd, lens, L):
    import torch
    c = Decode(lens, [min(L, n) for n in lens], heads, kv, hd)
    c.q *= 0.4  # scores of about one: thousands of keys count
    c.launch(G)
    torch.cuda.synchronize()
    k, v = values(*c.cache[:2]), values(*c.cache[2:])
    at = 0
    for s, n, m in zip(c.start, lens, c.L):
        seen = torch.arange(n, device="cuda")[None] <= (n - m + torch.arange(m, device="cuda"))[:, None]
        rounded_within(c.out[at:at + m], c.q[at:at + m].reshape(m, heads, hd), k[s:s + n], v[s:s + n], seen, 2.0 ** -11)
        at += m


@pytest.mark.parametrize("heads,kv,hd,lens,S,causal", [(24, 4, 256, [16], 4096, False), (24, 4, 256, [16, 5], 16384, True), (16, 2, 128, [1, 2], 9000, True), (4, 1, 64, [700, 900], 0, True),
                                                       (24, 4, 256, [40] * 40, 2048, False)])
def test_questions_whole_rows(G, heads, kv, hd, lens, S, causal):
    import torch
    c = Questions(lens, S, heads, kv, hd, causal, False)
    c.q *= 0.4
    c.launch(G)
    torch.cuda.synchronize()
    ks, vs = values(*c.cache[:2])[:S], values(*c.cache[2:])[:S]
    for a, b in list(zip(cu_of(lens), cu_of(lens)[1:]))[:4]:
        n = b - a
        k, v = (torch.cat((x, y[a:b].double().reshape(n, kv, hd))) for x, y in ((ks, c.k), (vs, c.v)))
        seen = torch.ones(n, S + n, dtype=torch.bool, device="cuda")
        if causal:
            seen[:, S:] = seen[:, S:].tril()
        rounded_within(c.out[a:b], c.q[a:b], k, v, seen, 2.0 ** -8)


# ---------------------------------------------------------------------------------------------
# sizes at the edge
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv,hd", [(192, 1, 64), (131, 1, 64), (256, 2, 128), (129, 1, 256)])
def test_more_query_heads_than_a_tile_has_rows(G, heads, kv, hd):
    """Groups above 128 heads: cut into equal parts where they divide, a head at a time where they do not."""
    for lens, S, causal in (([3, 40], 70, False), ([17], 0, True), ([5], 2000, True)):
        c = Questions(lens, S, heads, kv, hd, causal, True)
        c.launch(G)
        c.check()
    c = Decode([300, 5, 2000], [1, 2, 3], heads, kv, hd, gate=True)
    c.launch(G)
    c.check()


def test_new_tokens_of_empty_stretches_at_the_ends_of_the_cache(G):
    import torch
    c = Decode([0, 40, 0, 0], [1, 2, 3, 1], 24, 4, 256, max_len=64)
    c.t_start.copy_(torch.tensor([0, c.start[1], c.pool, c.pool]))
    c.launch(G)
    c.check()


def test_calls_without_an_error_word(G):
    import torch
    for c in (Questions([5, 30], 3000, 24, 4, 256, False, True), Decode([2000, 3], 2, 24, 4, 256)):
        keep = c.err
        c.err = None
        c.launch(G)
        c.err = keep
        c.check()
    q = Questions([5, 30], 300, 24, 4, 256, False, True)
    q.cu[1] = 99
    q.err = None
    q.launch(G)
    torch.cuda.synchronize()
    assert (q.out == -7.0).all()
