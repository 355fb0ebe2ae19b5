"""fb_linear_q4_decode refuses what it does not take before anything is launched. No GPU: addresses are made up."""
import ctypes

from fngine_b200 import lib as L


def call(lib, tokens=4, n=256, k=256, group=64, sdtype=L.DT_BF16, codes=0x100000, scales=0x200000, zeros=None, x=0x300000,
         kind=L.EPI_STORE_F32, out=0x400000, inj=None, gate=None, weight=True, epilogue=True):
    w = L.Q4Weight(codes, scales, zeros, sdtype, group, n, k)
    e = L.LinearEpilogue(kind, 0, out, inj, gate)
    st = lib.fb_linear_q4_decode(x, tokens, ctypes.byref(w) if weight else None, ctypes.byref(e) if epilogue else None, None)
    return st, lib.fb_last_error_string()


def test_refusals(fb_built):
    lib = L.load()
    for bad, word in [(dict(tokens=0), b"1..16"), (dict(tokens=17), b"1..16"), (dict(tokens=-1), b"1..16"), (dict(k=192), b"k % 128"),
                      (dict(k=0), b"shape"), (dict(n=0), b"shape"), (dict(n=-8), b"shape"), (dict(group=16), b"groups"), (dict(group=256), b"groups"),
                      (dict(group=0), b"groups"), (dict(n=2 ** 25, k=2048, group=32), b"2^31"), (dict(sdtype=7), b"scales"), (dict(kind=5), b"epilogue"), (dict(kind=-1), b"epilogue"),
                      (dict(kind=L.EPI_GR_WRITE), b"inj"), (dict(kind=L.EPI_SHARED_SCALE), b"gate_logit"), (dict(kind=L.EPI_SWIGLU, n=33), b"SwiGlu"),
                      (dict(codes=0x100008), b"aligned"), (dict(scales=0x200002), b"aligned"), (dict(zeros=0x500001), b"aligned"),
                      (dict(x=0x300008), b"aligned"), (dict(out=0x400002), b"aligned"), (dict(out=0x400001, kind=L.EPI_STORE_BF16), b"aligned"),
                      (dict(out=0x300400), b"memory of x"), (dict(out=0x2ffff0), b"memory of x"), (dict(x=None), b"null"), (dict(out=None), b"null"),
                      (dict(codes=None), b"null"), (dict(scales=None), b"null"), (dict(weight=False), b"null"), (dict(epilogue=False), b"null")]:
        st, msg = call(lib, **bad)
        assert st == 1 and word in msg, (bad, st, msg)
