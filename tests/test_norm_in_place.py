"""The stream's rows in place of x's are taken with x's stride alone: with another one, rows would be written over before
they are read.  Reported before any device call."""
import ctypes as C

from helpers import pkg

FAKE = 1 << 20  # never dereferenced


def test_y_in_place_of_x_has_its_stride():
    L = pkg().lib()
    for stride_x, stride_y in ((8, 16), (16, 8)):
        o = pkg().NormGateOption(dim=8, postNorm=0, preNorm=0, gateRows=0, residualScale=1.0, blockScale=1.0, epsilon=1e-6,
                                 dataType=0, strideX=stride_x, strideF=8, strideGate=8, strideY=stride_y, strideH=8)
        L.launchNormGateResidual(C.byref(o), FAKE, None, None, None, None, None, None, FAKE, None, 4, None)
        assert L.tinymlp_last_error() and "stride" in L.tinymlp_last_error_message().decode()
