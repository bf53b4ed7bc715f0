"""Limits of the operators of requests in pages that Python and the header both state."""
import os
import re

from dtas_amd import _lib


def test_the_headers_limit_is_the_librarys():
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(_lib.__file__))), "include", "dtas_abi.h")) as f:
        assert int(re.search(r"#define DTAS_MAX_BEAMS (\d+)", f.read()).group(1)) == _lib.MAX_BEAMS
    call = lambda name, *args: (getattr(_lib.lib(), name)(*args), _lib.last_error())
    at = [0x10000000 * (i + 1) for i in range(10)]  # never dereferenced: the calls end before a launch
    for beams, refused in ((_lib.MAX_BEAMS, False), (_lib.MAX_BEAMS + 1, True)):
        for rc, message in (call("dtas_beam_select_f32", *at[:7], 0, beams, 100, 0, None),
                            call("dtas_page_reorder_f16", *at[:4], at[4], *at[5:7], at[4], *at[8:], 2, 0, beams, 5, 2, 64, 16, 40, None)):
            assert (rc, f"up to {_lib.MAX_BEAMS} beams" in message) == ((-1, True) if refused else (0, False))
