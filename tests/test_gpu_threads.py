"""Drafted sampling while another thread uses the GPU.  On this runtime a copy through the legacy stream (hipMemcpy) or a
hipDeviceSynchronize, made by any thread while a stream is being captured, fails, and the capture can be neither used nor ended: so the
call captures nothing."""
import ctypes
import threading

import numpy as np
import pytest

from test_gpu_sample_drafted import O, decoder, features, small, stattn_mod      # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


class LegacyCopies(object):
    """A thread that copies through the legacy stream all the time; `failed` counts the copies that were refused."""

    def __enter__(self):
        hip = ctypes.CDLL("libamdhip64.so")
        buf, host = ctypes.c_void_p(), ctypes.create_string_buffer(4096)
        assert hip.hipMalloc(ctypes.byref(buf), ctypes.c_size_t(4096)) == 0
        self.failed, self.copies, self.go = 0, 0, True

        def loop():
            while self.go:
                self.failed += hip.hipMemcpy(buf, host, ctypes.c_size_t(4096), 1) != 0
                self.copies += 1
            hip.hipGetLastError()
            hip.hipFree(buf)
        self.thread = threading.Thread(target=loop)
        self.thread.start()
        return self

    def __exit__(self, *exc):
        self.go = False
        self.thread.join()


def test_drafted_sampling_beside_another_threads_copies(stattn_mod, O):      # noqa: F811
    """Thirty calls of different shapes: no copy of the other thread fails, and the results are those of an undisturbed handle."""
    opt, P = small(O)
    b = O.synthetic_batch(opt, B=3, T=5, K=3, t=3, seed=81)

    def call(dec, maxlen):
        u = np.random.RandomState(maxlen).random_sample((maxlen, 5, 3)).astype(np.float32)
        return dec.sample_drafted(*features(b), draft=2, maxlen=maxlen, uniforms=np.minimum(u, np.float32(1 - 2.0 ** -24)))
    quiet, dec = decoder(stattn_mod, opt, P), decoder(stattn_mod, opt, P)
    want = [call(quiet, n) for n in range(1, 31)]
    with LegacyCopies() as other:
        got = [call(dec, n) for n in range(1, 31)]
    assert got == want
    assert other.copies > 30 and other.failed == 0


def test_calls_beside_an_open_capture(stattn_mod, O):      # noqa: F811
    """This thread captures a stream; another one makes and uses handles meanwhile.  Neither disturbs the other: the calls go through, and
    the capture ends as a graph."""
    opt, P = small(O)
    b = O.synthetic_batch(opt, B=3, T=5, K=3, t=3, seed=83)
    u = np.random.RandomState(1).random_sample((6, 5, 3)).astype(np.float32)

    def calls():
        dec = decoder(stattn_mod, opt, P)
        dec.set_seed(4)
        out = [dec.sample_drafted(*features(b), draft=2, maxlen=6, uniforms=u), dec.sample_search(*features(b), maxlen=6)]
        g, gm, l, m = (b[k][0] for k in ('ctxg', 'mask_ctxg', 'ctxl', 'ctxm'))
        _, h, c = dec.f_init(g, gm)
        out.append([np.asarray(a).tolist() for a in dec.f_next(np.array([-1]), g, gm, l, None, m, None, h[None], c[None])])
        return out + [{k: dec.get_param(k).tolist() for k in ('ff_logit_W', 'ff_logit_b')}]
    want, got = calls(), []
    hip = ctypes.CDLL("libamdhip64.so")
    buf, stream, graph = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipMalloc(ctypes.byref(buf), ctypes.c_size_t(8192)) == 0 and hip.hipStreamCreateWithFlags(ctypes.byref(stream), 1) == 0

    def copy():
        return hip.hipMemcpyAsync(ctypes.c_void_p(buf.value + 4096), buf, ctypes.c_size_t(4096), 3, stream)
    assert hip.hipStreamBeginCapture(stream, 1) == 0 and copy() == 0        # 1: this thread's calls are the capture's, other threads' are not
    thread = threading.Thread(target=lambda: got.append(calls()))
    thread.start()
    thread.join()
    last, end = copy(), hip.hipStreamEndCapture(stream, ctypes.byref(graph))
    assert got == [want]
    assert (last, end) == (0, 0) and graph.value
    assert hip.hipGraphDestroy(graph) == 0 and hip.hipStreamDestroy(stream) == 0 and hip.hipFree(buf) == 0
