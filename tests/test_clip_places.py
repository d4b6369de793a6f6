"""Where results and norms of hctr_clip_gradients may lie: what is refused before anything is launched."""
import os

import pytest

from hetuctr_amd import build, capi

pytestmark = pytest.mark.skipif(not os.path.exists(build.LIB), reason="needs the built library")
FAR = 1 << 30


@pytest.mark.parametrize("gradients, norm, given", [
    ([(65536, 65536, 9, capi.F32)], 0, 65536),                      # the norm that is given is a value of a result
    ([(65536, 65536, 9, capi.F32)], 0, 65536 + 32),                 # its last one
    ([(65536, FAR, 9, capi.F32)], 0, FAR + 4),
    ([(65536, 65536, 9, capi.BF16)], 0, 65536 + 16),                # half of the norm
    ([(65536, 65536, 9, capi.F32)], 65536 + 8, 0),                  # the norm that is made is written to a result
    ([(65536, FAR, 9, capi.F32)], 65536 + 8, 0),                    # or to a gradient
    ([(65536, 65536, 9, capi.F32), (FAR, FAR, 5, capi.F32)], FAR + 16, 4096),
    ([(65536, 65536, 9, capi.F32)], 4096, 4098)])                   # two norms that overlap
def test_norms_in_the_way_are_refused(gradients, norm, given):
    need = capi.clip_gradients(gradients, 1.0, norm, given, (0, 0), space=True)
    with pytest.raises(RuntimeError, match="lies where"):
        capi.clip_gradients(gradients, 1.0, norm, given, (1 << 20, need))


def test_norms_beside_results_are_not():
    # (the workspace that is missing is what these calls are refused for, or there is nothing to do)
    for gradients, norm, given in (([(65536, 65536, 9, capi.F32)], 65536 + 36, 0), ([(65536, FAR, 9, capi.F32)], 65536 - 4, 0), ([(65536, FAR, 9, capi.F32)], FAR - 4, 0)):
        with pytest.raises(RuntimeError, match="workspace"):
            capi.clip_gradients(gradients, 1.0, norm, given, (0, 0))
    capi.clip_gradients([], 1.0, 4096, 4096, (0, 0))                # one norm, given and returned
