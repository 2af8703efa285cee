"""What the low-precision attention layer's entry points refuse, before anything reaches a GPU: DCD_E_INVALID and no launch."""
import ctypes as C

import pytest

BUF = C.c_void_p(0x10000)      # never dereferenced: every call below is refused on its arguments
ODD = C.c_void_p(0x10008)


def refused(dcd, name, args):
    from decidra_b200 import _lib
    return getattr(_lib.load(), name)(*args) == _lib.E_INVALID


def with_each(base, changes):
    for key, value in changes:
        args = dict(base)
        args[key] = value
        yield key, list(args.values())


NORM = dict(x=BUF, xs=64, w=BUF, out=BUF, scales=BUF, rows=2, cols=64, eps=1e-6, zc=1, clip=1.0, rt=0, dtype=1, st=None)
ADD = dict(x=BUF, xs=64, mix=C.c_void_p(0x20000), ms=64, w=BUF, res=C.c_void_p(0x30000), out=BUF, scales=BUF, rows=2, cols=64, eps=1e-6, zc=1, clip=1.0, rt=0, dtype=1, st=None)


@pytest.mark.parametrize("base,name", [(NORM, "dcd_k_rmsnorm_fp8"), (ADD, "dcd_k_add_rmsnorm_fp8")])
def test_norm_refusals(dcd, base, name):
    changes = [("x", None), ("w", None), ("out", None), ("scales", None), ("rows", -1), ("cols", 0), ("cols", -8), ("xs", 63), ("dtype", 2), ("dtype", -1)]
    if base is ADD:
        changes += [("mix", None), ("res", None), ("ms", 10)]
    for key, args in with_each(base, changes):
        assert refused(dcd, name, args), key
    if base is ADD:  # in place only where a row is written where it was read
        for a in ({"res": BUF, "xs": 128}, {"res": C.c_void_p(0x20000), "ms": 72}):
            assert refused(dcd, name, list({**ADD, **a}.values()))


WRITE = dict(k=BUF, ks=128, v=BUF, vs=128, slots=None, kc=BUF, ksc=BUF, vc=BUF, vsc=BUF, total=10, rows=4, kv=2, hd=64, dtype=1, err=None, st=None)
READ = dict(kc=BUF, ksc=BUF, vc=BUF, vsc=BUF, total=10, slots=None, k=BUF, v=BUF, rows=4, kv=2, hd=64, dtype=1, err=None, st=None)


def test_cache_refusals(dcd):
    common = [("k", None), ("v", None), ("kc", None), ("ksc", None), ("vc", None), ("vsc", None), ("kc", ODD), ("vsc", ODD), ("rows", -1), ("rows", 11), ("kv", 0),
              ("hd", 96), ("hd", 0), ("dtype", 3)]
    for key, args in with_each(WRITE, common + [("ks", 127), ("vs", 0)]):
        assert refused(dcd, "dcd_k_kv4_write", args), key
    for key, args in with_each(READ, common + [("k", ODD), ("v", ODD)]):
        assert refused(dcd, "dcd_k_kv4_read", args), key


QUESTIONS = dict(q=BUF, qs=1024, k=BUF, ks=256, v=BUF, vs=256, kc=BUF, ksc=BUF, vc=BUF, vsc=BUF, S=100, gate=None, gs=0, out=BUF, cu=BUF, B=2, T=9, heads=8, kv=2, hd=128,
                 causal=0, ws=BUF, wb=1 << 40, err=None, st=None)
DECODE = dict(q=BUF, qs=1024, kc=BUF, ksc=BUF, vc=BUF, vsc=BUF, total=1000, start=BUF, len=BUF, max_len=100, gate=None, gs=0, out=BUF, cu=BUF, B=2, T=2, heads=8, kv=2, hd=128,
              ws=BUF, wb=1 << 40, err=None, st=None)


def test_attention_refusals(dcd):
    from decidra_b200 import _lib
    common = [("q", None), ("q", ODD), ("qs", 1023), ("qs", 1028), ("kc", None), ("ksc", None), ("vc", ODD), ("vsc", None), ("out", None), ("out", ODD), ("cu", None),
              ("B", 0), ("B", -1), ("T", 0), ("heads", 0), ("heads", 7), ("kv", 0), ("kv", 3), ("hd", 96), ("hd", 512), ("hd", 32)]
    for key, args in with_each(QUESTIONS, common + [("k", None), ("v", ODD), ("ks", 255), ("vs", 260), ("S", -1)]):
        assert refused(dcd, "dcd_k_attention_kv4", args), key
    for key, args in with_each(DECODE, common + [("start", None), ("len", None), ("max_len", -1)]):
        assert refused(dcd, "dcd_k_attention_kv4_decode", args), key
    for base, name in ((QUESTIONS, "dcd_k_attention_kv4"), (DECODE, "dcd_k_attention_kv4_decode")):
        assert refused(dcd, name, list({**base, "gate": BUF, "gs": 2047}.values()))
        assert refused(dcd, name, list({**base, "gate": ODD, "gs": 2048}.values()))
        assert refused(dcd, name, list({**base, "gate": BUF, "gs": (1 << 24) + 8}.values()))
    lib = _lib.load()
    for base, name, n in ((QUESTIONS, "dcd_k_attention_kv4", "S"), (DECODE, "dcd_k_attention_kv4_decode", "max_len")):
        size = getattr(lib, name + "_workspace")
        need = size(base["B"], base["T"], base[n], base["heads"], base["kv"], base["hd"])
        if need:
            for a in ({"ws": None}, {"wb": need - 1}, {"ws": ODD}):
                assert refused(dcd, name, list({**base, **a}.values())), a
        # no size for a shape that the call refuses
        for bad in ((0, 9, 100, 8, 2, 128), (2, 0, 100, 8, 2, 128), (2, 9, -1, 8, 2, 128), (2, 9, 100, 7, 2, 128), (2, 9, 100, 8, 2, 96)):
            assert size(*bad) == 0


def test_pointers_off_their_elements_are_refused(dcd):
    """On the device they would be misaligned addresses. Each operand two bytes off, or one (bf16), or four (64-bit integers)."""
    def off(n):
        return C.c_void_p(0x10000 + n)

    for dtype, step in ((0, 2), (0, 1), (1, 1)):
        for base, name, keys in ((NORM, "dcd_k_rmsnorm_fp8", "x w"), (ADD, "dcd_k_add_rmsnorm_fp8", "x mix w res"), (WRITE, "dcd_k_kv4_write", "k v")):
            for key, args in with_each({**base, "dtype": dtype}, [(key, off(step)) for key in keys.split()]):
                assert refused(dcd, name, args), (name, key)
    for base, name, keys in ((NORM, "dcd_k_rmsnorm_fp8", "scales"), (ADD, "dcd_k_add_rmsnorm_fp8", "scales"), (WRITE, "dcd_k_kv4_write", "err slots"),
                             (READ, "dcd_k_kv4_read", "err slots"), (QUESTIONS, "dcd_k_attention_kv4", "cu err"), (DECODE, "dcd_k_attention_kv4_decode", "cu len start err")):
        for key, args in with_each(base, [(key, off(2)) for key in keys.split()]):
            assert refused(dcd, name, args), (name, key)
    for base, name, key in ((WRITE, "dcd_k_kv4_write", "slots"), (READ, "dcd_k_kv4_read", "slots"), (DECODE, "dcd_k_attention_kv4_decode", "start")):
        assert refused(dcd, name, list({**base, key: off(4)}.values())), (name, key)


def test_no_rows_need_no_arrays(dcd):
    """Arrays of no elements have no address: rows 0 does nothing and succeeds, whatever the sizes that are checked allow."""
    from decidra_b200 import _lib
    for base, name, arrays in ((NORM, "dcd_k_rmsnorm_fp8", "x out scales"), (ADD, "dcd_k_add_rmsnorm_fp8", "x mix res out scales"), (WRITE, "dcd_k_kv4_write", "k v"),
                               (READ, "dcd_k_kv4_read", "k v"), (WRITE, "dcd_k_kv4_write", "k v kc ksc vc vsc"), (READ, "dcd_k_kv4_read", "k v kc ksc vc vsc")):
        args = {**base, "rows": 0, **{key: None for key in arrays.split()}}
        assert getattr(_lib.load(), name)(*args.values()) == 0, name
        assert refused(dcd, name, list({**args, "dtype": 2}.values())), name


def test_new_tokens_workspace_is_bounded(dcd):
    """A bound far above the lengths and many tokens of one sequence both cost next to nothing; a call of one token asks for little."""
    from decidra_b200 import _lib
    size = _lib.load().dcd_k_attention_kv4_decode_workspace
    assert size(64, 64, 1 << 30, 24, 4, 256) == size(64, 64, 20000, 24, 4, 256) < 64 << 20
    assert size(1, 2000, 100_000, 24, 4, 256) < 64 << 20
    assert size(1, 2000, 100_000, 16, 1, 128) < 128 << 20
    assert size(1, 1, 2048, 24, 4, 256) < 8 << 20
    # what is enough for the largest call is enough for every smaller one
    for heads, kv, hd in ((24, 4, 256), (16, 2, 128), (4, 1, 64), (15, 3, 256)):
        largest = size(64, 300, 20000, heads, kv, hd)
        for B, T, n in ((64, 64, 20000), (1, 300, 20000), (1, 1, 20000), (2, 8, 777), (64, 300, 1), (9, 36, 8192), (1, 4, 16384)):
            assert size(B, T, n, heads, kv, hd) <= largest
