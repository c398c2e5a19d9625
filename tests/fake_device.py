"""Checks of libmimoe.so's host code against a HIP runtime of host memory (cpp/fake_hip.cpp), in which allocations can
fail and kernels are counted, not run.  A program of its own, without torch: the runtime has to be loaded before the
library.  Usage: fake_device.py <fake runtime> <library> <check>; prints ok."""
import ctypes
import sys

P, I64, I, F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
Q8_0, Q4_0, W4A16, MXFP4 = range(4)
BF16, F32 = 1, 2
EHIP = 4
STREAM = P(1 << 20)      # a stream of the caller's, which does not wait for the default one
DATA = ctypes.create_string_buffer(1 << 22)   # what every argument points to; only host sources are read
AT = P((ctypes.addressof(DATA) + 255) & ~255)
SHAPE = {Q8_0: (4, 128, 64), Q4_0: (4, 128, 64), W4A16: (2, 512, 128), MXFP4: (4, 192, 96)}

ARGS = {
    "mi_moe_create": [I64, I64, I64, I, ctypes.POINTER(P)], "mi_moe_destroy": [P], "mi_moe_reserve": [P, I64, I64, P],
    "mi_moe_store_mxfp4": [P, P, P, P, P, I, P], "mi_moe_store_quantized": [P, P, P, P, P, I, I, P],
    "mi_moe_store_awq": [P, P, P, P, P, P, P, I64, I, I, P],
    "mi_moe_quantize_and_store_expert": [P, I64, I, P, I, I, P],
    "mi_moe_hybrid_create": [I64, I64, I64, I, P, I, ctypes.POINTER(P)], "mi_moe_hybrid_destroy": [P],
    "mi_moe_hybrid_store_quantized": [P, P, P, P, P, I, I, P], "mi_moe_hybrid_forward": [P, P, P, P, P, I64, I64, I, P],
    "mi_moe_forward_noalloc": [P, P, P, P, P, I64, I64, I, P],
    "mi_moe_forward": [P, P, P, P, P, I64, I64, I, P],
    "mi_moe_forward_logits": [P, P, P, P, I, I64, I64, I, I, P, P, P],
    "mi_moe_forward_scores": [P, P, P, P, I, I64, I64, P, I, I64, I64, I64, I, F, I, P, P, P],
}


class Device:
    def __init__(self, fake, lib):
        self.f = ctypes.CDLL(fake, mode=ctypes.RTLD_GLOBAL)
        self.f.fake_mallocs.restype = self.f.fake_launches.restype = self.f.fake_live.restype = ctypes.c_long
        self.f.fake_fail_at.argtypes = [ctypes.c_long]
        self.lib = ctypes.CDLL(lib)
        self.lib.mi_moe_last_error.restype = ctypes.c_char_p
        for name, args in ARGS.items():
            getattr(self.lib, name).argtypes = args

    def call(self, name, *args):
        return getattr(self.lib, "mi_moe_" + name)(*args)

    def ok(self, name, *args):
        rc = self.call(name, *args)
        assert rc == 0, (name, rc, self.lib.mi_moe_last_error())

    def handle(self, quant):
        h = P()
        self.ok("create", *SHAPE[quant], quant, ctypes.byref(h))
        return h

    def live(self):
        """The sizes of all allocations, and which were cleared as a whole."""
        sizes, cleared = (ctypes.c_size_t * 256)(), (I * 256)()
        n = self.f.fake_live(sizes, cleared, 256)
        return sorted((sizes[i], cleared[i]) for i in range(n))

    # calls of each kind, the same for every handle
    def store(self, h, quant):
        if quant == MXFP4:
            return self.call("store_mxfp4", h, AT, AT, AT, AT, 1, STREAM)
        if quant == W4A16:
            return self.call("store_awq", h, *[AT] * 6, 128, BF16, 1, STREAM)
        return self.call("store_quantized", h, AT, AT, AT, AT, BF16, 1, STREAM)

    def online(self, h, quant):
        return self.call("quantize_and_store_expert", h, 1, 2, AT, F32, 1, STREAM)

    def logits(self, h, T, K=2, ldt=F32, act=BF16, x=AT, y=AT, logits=AT):
        return self.call("forward_logits", h, x, y, logits, ldt, T, K, 1, act, None, None, STREAM)

    def scores(self, h, T, K=2, ldt=F32, act=BF16, x=AT, y=AT, logits=AT):
        return self.call("forward_scores", h, x, y, logits, ldt, T, K, None, 1, 1, 1, 1, 1, 1.0, act, None, None, STREAM)

    def forward(self, h, T, K=2):
        return self.call("forward", h, AT, AT, AT, AT, T, K, BF16, STREAM)


def retried(d, quant, before, call, after, first=None):
    """call fails at each of its allocations in turn; `after` on such a handle leaves what it leaves on one where the
    call was never made.  first: only so many allocations."""
    def run(fail):
        h = d.handle(quant)
        before(h)
        n = None
        if fail is not None:
            d.f.fake_fail_at(fail)
            rc = call(h)
            n = d.f.fake_mallocs()
            d.f.fake_fail_at(-1)
            if n <= fail:            # it has no allocation of that number
                assert rc == 0
                d.ok("destroy", h)
                return None
            assert rc == EHIP and b"out of memory" in d.lib.mi_moe_last_error(), (rc, d.lib.mi_moe_last_error())
            assert d.f.fake_last_error() == 0, "the caller's next check of a launch reports it"
        rc = after(h)
        assert rc == 0, (fail, rc, d.lib.mi_moe_last_error())
        left = d.live()
        d.ok("destroy", h)
        assert d.live() == [], "allocations left behind a handle"
        return left
    want, tried = run(None), 0
    while tried != first:
        got = run(tried)
        if got is None:
            break
        assert got == want, (tried, got, want)
        tried += 1
    return tried


def weights(d):
    for quant in (Q8_0, Q4_0, W4A16, MXFP4):
        store = lambda h: d.store(h, quant)
        assert retried(d, quant, lambda h: None, store, store) == 4, quant
        if quant in (Q8_0, MXFP4):
            online = lambda h: d.online(h, quant)
            assert retried(d, quant, lambda h: None, online, online) == 4, quant
    # weights stored a second time, with no memory to be had: the handle serves on
    for quant in (Q8_0, Q4_0, W4A16, MXFP4):
        h = d.handle(quant)
        assert d.store(h, quant) == 0
        have = d.live()
        d.f.fake_fail_at(0)
        assert d.store(h, quant) == 0 and d.f.fake_mallocs() == 0, quant
        d.f.fake_fail_at(-1)
        assert d.live() == have
        d.ok("destroy", h)


def workspace(d):
    for quant in (Q8_0, Q4_0, W4A16, MXFP4):
        for first in (None, 1, 20):       # calls before the one that fails
            def before(h):
                assert d.store(h, quant) == 0
                if first:
                    assert d.forward(h, first) == 0
            tried = retried(d, quant, before, lambda h: d.forward(h, 400), lambda h: d.forward(h, first or 1))
            assert tried >= 7, (quant, first, tried)


def picks(d):
    for quant in (Q4_0, W4A16, MXFP4):
        for call in (d.logits, d.scores):
            def before(h):
                assert d.store(h, quant) == 0 and call(h, 1) == 0
            assert retried(d, quant, before, lambda h: call(h, 2000), lambda h: call(h, 1), first=2) == 2


def refused(d):
    odd = P(AT.value + 8)
    for quant in (Q4_0, W4A16, MXFP4):
        for call in (d.logits, d.scores):
            h = d.handle(quant)
            have, done = d.live(), (d.f.fake_launches(), d.f.fake_syncs())
            assert call(h, 4096) == 2, "weights not stored"

            def nothing_done(rc, word):
                assert rc == 1 and word in d.lib.mi_moe_last_error(), (quant, rc, d.lib.mi_moe_last_error())
                assert d.live() == have and (d.f.fake_launches(), d.f.fake_syncs()) == done, (quant, word)
            assert d.live() == have and (d.f.fake_launches(), d.f.fake_syncs()) == done
            assert d.store(h, quant) == 0
            have, done = d.live(), (d.f.fake_launches(), d.f.fake_syncs())
            nothing_done(call(h, 1 << 24), b"too large")
            nothing_done(call(h, 4096, act=7), b"fp16 or bf16")
            nothing_done(call(h, 4096, ldt=7), b"logits dtype")
            nothing_done(call(h, 4096, K=SHAPE[quant][0] + 1), b"top_k")
            nothing_done(call(h, 4096, logits=None), b"null")
            nothing_done(call(h, 4096, x=None), b"null")
            nothing_done(call(h, 4096, y=None), b"null")
            nothing_done(call(h, 4096, x=odd), b"aligned")
            assert call(h, 0) == 0 and call(h, 4096) == 0
            d.ok("destroy", h)


def clears(d):
    """fake_unordered counts launches while a clear on the default stream may still be running."""
    for quant in (Q8_0, Q4_0, W4A16, MXFP4):
        h = d.handle(quant)
        assert d.store(h, quant) == 0 and d.f.fake_unordered() == 0, ("stored", quant)
        assert d.forward(h, 1) == 0 and d.f.fake_unordered() == 0, ("forward", quant)
        d.ok("destroy", h)
        if quant in (Q8_0, MXFP4):
            h = d.handle(quant)
            assert d.online(h, quant) == 0 and d.f.fake_unordered() == 0, ("online", quant)
            d.ok("destroy", h)


def mx_workspace(d):
    """What an MXFP4 layer reads: packets of 32 bytes a block (rows in whole 128s), fp32 outputs, routing; no block
    scales beside them."""
    E, H, I_ = SHAPE[MXFP4]
    h = d.handle(MXFP4)
    assert d.store(h, MXFP4) == 0
    have = d.live()
    d.ok("reserve", h, 512, 2, STREAM)
    new = d.live()
    for b in have:
        new.remove(b)
    big = sorted(b[0] for b in new if b[0] > 8192)
    assert big == sorted([1024 * 128, 512 * 256, 1024 * H * 4]), big   # intermediate, hidden rows, outputs
    assert not any(b[0] in (1024 * I_ // 32 * 4, 512 * H // 32 * 4) for b in new), new
    d.ok("destroy", h)
    # 7000 rows of I = 4096 fit the array of the call without allocation: 4096 + 256 + 128 bytes each, and routing
    h = P()
    d.ok("create", 2, 64, 4096, MXFP4, ctypes.byref(h))
    assert d.store(h, MXFP4) == 0
    assert d.call("forward_noalloc", h, AT, AT, AT, AT, 7000, 1, BF16, STREAM) == 0, d.lib.mi_moe_last_error()
    assert d.call("forward_noalloc", h, AT, AT, AT, AT, 7600, 1, BF16, STREAM) == 1
    d.ok("destroy", h)


def hybrid_handle(d, quant=Q4_0):
    mask, h = (ctypes.c_uint8 * 4)(1, 0, 1, 0), P()
    d.ok("hybrid_create", *SHAPE[quant], quant, mask, 1, ctypes.byref(h))
    d.ok("hybrid_store_quantized", h, AT, AT, AT, AT, BF16, 0, STREAM)
    return h


def hybrid_leaves_nothing(d):
    for quant in (Q8_0, Q4_0):
        d.ok("hybrid_destroy", hybrid_handle(d, quant))
        assert d.live() == [], d.live()


def hybrid_staging(d):
    forward = lambda h, T: d.call("hybrid_forward", h, AT, AT, AT, AT, T, 2, BF16, STREAM)

    def left(fail):   # a call, one that fails to grow, and one that fits what the first left
        h = hybrid_handle(d)
        assert forward(h, 1) == 0
        d.f.fake_fail_at(fail)
        assert fail < 0 or forward(h, 400) == EHIP
        assert d.f.fake_last_error() == 0
        d.f.fake_fail_at(-1)
        assert forward(h, 1) == 0
        sizes = d.live()
        d.ok("hybrid_destroy", h)
        return sizes
    want = left(-1)
    for fail in range(5):   # the staging buffers; the device handle's workspace is not reached
        got = left(fail)
        assert got == want, (fail, got, want)


CHECKS = {f.__name__: f for f in (weights, workspace, picks, refused, clears, mx_workspace, hybrid_leaves_nothing, hybrid_staging)}

if __name__ == "__main__":
    CHECKS[sys.argv[3]](Device(sys.argv[1], sys.argv[2]))
    print("ok")
