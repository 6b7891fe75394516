"""CPU checks of what the adapters refuse before any device work."""
from __future__ import annotations

import pytest

from test_lora_blocks_cpu import lora_desc, refused


@pytest.mark.parametrize("f", ["b2g_lora_up", "b2g_lora"])
@pytest.mark.parametrize("which", ["y", "out"])
def test_addresses_between_elements(f, which):
    """Rows may begin anywhere, elements may not."""
    import b2g

    lib = b2g.load()
    for y_dtype, places in ((b2g.BF16, (257, 263)), (b2g.F32, (257, 258, 262))):
        for at in places:
            refused(lib, getattr(lib, f)(lora_desc(y_dtype=y_dtype, **{which: at}), None), 2, f"{f}: y and out")


def test_sizes_are_refused_before_the_first_half_runs():
    """lora_up's launch would not fit a grid: lora says so too, not lora_down's launch before it."""
    import b2g

    lib = b2g.load()
    for f in ("b2g_lora_up", "b2g_lora"):
        refused(lib, getattr(lib, f)(lora_desc(rows=2 ** 30, N=2 ** 20, ldy=2 ** 20, ldo=2 ** 20), None), 2, f"{f}: size")
