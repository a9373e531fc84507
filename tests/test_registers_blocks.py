"""Registers that the kernels of decoder layers spill (see test_registers.py)."""
import re

import pytest

from test_registers import spills  # noqa: F401 (a fixture)


@pytest.mark.parametrize("kernel", [
    r"k_block_(skinny|tile)I",         # every form
    r"k_(join_parts|align_rows|quantize_rows|quantize_tiles|rotary)",
    r"k_cache_promptILi(2|4)E",        # heads of 64 and 128
    r"k_cache_attentionI.*Lb1EEE",     # few rows
    r"k_cache_(append|join|join_rows)I",
])
def test_kernels_spill_no_registers(spills, kernel):  # noqa: F811
    forms = {n: s for n, s in spills.items() if re.search(kernel, n)}
    assert forms and max(forms.values()) == 0, {n: s for n, s in forms.items() if s}
