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
