"""A 4-bit cache whose planes overlap is refused by what writes to it, before the device is needed."""
import ctypes

import pytest

import g4hip


@pytest.mark.parametrize("i", range(4))
@pytest.mark.parametrize("j", range(4))
def test_append_to_planes_that_overlap(i, j):
    # 7 rows of 256 in use: 896 bytes of codes (k, v), 112 of scales
    planes, size = [1 << 20, 2 << 20, 3 << 20, 4 << 20], (896, 896, 112, 112)
    for at in (planes[j], planes[j] + size[j] - 16) if i != j else ():
        p = list(planes)
        p[i] = at
        cache = ctypes.byref(g4hip.Kv4(*p, 100, 256))
        assert g4hip.lib().g4_kv4_append(cache, 16 << 20, 17 << 20, 4, 3) == g4hip.G4_E_ARG
        assert "planes overlap" in g4hip.lib().g4_last_error().decode()
