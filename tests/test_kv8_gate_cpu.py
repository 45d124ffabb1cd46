"""What ta_kv8_gate_append refuses before it launches anything.  CPU only."""
import ctypes

from treeattn_amd import _lib


def test_refused_arguments():
    L = _lib.lib()
    P = 4096      # never dereferenced
    c = ctypes.byref(_lib.Kv8(P, P, P, 8, 4, 10, P, 4096, 2048, P, 2, 4, 64))

    def call(cache=c, D=64, t=P, n=1, levels=True, blevel=4, arity=1, q=0.5, dtype=2, lg=P):
        p = (ctypes.c_void_p * 2)(P, P)
        s = (ctypes.c_int64 * 2)(64, 64)
        bl = (ctypes.c_int32 * 2)(blevel, blevel + 1)
        at = [p, (ctypes.c_void_p * 2)(lg, P), p] if levels else [None] * 3
        return L.ta_kv8_gate_append(cache, dtype, 1, 2, D, t, n, *at, s, s, bl, arity, q, None)

    def refused(rc, text, code=1):
        assert rc == code and text in L.ta_last_error(), (rc, L.ta_last_error())
    refused(call(cache=None), b'bad cache description')
    refused(call(D=48), b'head dim', 2)
    refused(call(t=None), b'bad arguments')
    refused(call(arity=5), b'bad arguments')
    refused(call(q=1.5), b'bad arguments')
    refused(call(n=33), b'bad arguments')
    refused(call(dtype=9), b'dtype')
    refused(call(levels=False), b'levels without')
    refused(call(blevel=5), b'leaf blocks')
    refused(call(lg=None), b'log sums')
    assert call(n=0) == 0
