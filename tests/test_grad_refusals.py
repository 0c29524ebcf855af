"""Where the gradients' norm may be (include/grad_abi.h): refused before any device call (no GPU)."""
import pytest

from test_serving_refusals import FAKE, error, tensors


@pytest.mark.parametrize("items,norm", [
    ([(FAKE, None, 8, 0)], FAKE), ([(FAKE, None, 8, 0)], FAKE + 28), ([(FAKE, FAKE + 64, 8, 0)], FAKE + 92),
    ([(FAKE + 512, None, 1, 1), (FAKE + 256, FAKE + 2, 3, 1)], FAKE + 4), ([(FAKE, FAKE, 1, 2)], FAKE)])
def test_a_norm_within_what_is_written(items, norm):
    t = tensors(*items)
    assert "overlaps" in error("launchGradClip", t, len(items), 1.0, 0, norm, None)
    assert "overlaps" in error("launchGradNormClip", t, len(items), 0, 1.0, 1.0, 0, norm, None)


@pytest.mark.parametrize("norm", [FAKE, FAKE + 28])
def test_a_norm_within_what_is_read(norm):
    """It may not be written while clipping reads that."""
    t = tensors((FAKE, FAKE + 64, 8, 0))
    assert "overlaps" in error("launchGradNormClip", t, 1, 0, 1.0, 1.0, 0, norm, None)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_a_norm_off_its_alignment(off):
    t = tensors((FAKE + 64, None, 8, 0))
    assert "aligned" in error("launchGradNorm", t, 1, 0, 1.0, FAKE + off, None)
    assert "aligned" in error("launchGradClip", t, 1, 1.0, 0, FAKE + off, None)
    assert "aligned" in error("launchGradNormClip", t, 1, 0, 1.0, 1.0, 0, FAKE + off, None)


def test_a_norm_beside_tensors():
    """Nothing to do, so nothing is launched: tensors of no elements overlap nothing."""
    t = tensors((FAKE, None, 0, 0), (FAKE + 4, FAKE + 4, 0, 1))
    assert error("launchGradClip", t, 2, 1.0, 0, FAKE, None) == ""
