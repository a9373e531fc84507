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


@pytest.mark.parametrize("kernel,most", [
    (r"k_cache_promptILi8E", 21),                  # heads of 256
    (r"k_cache_attentionIfLi4ELi2ELb0E", 45),      # rows a column: f32, 128 elements, two tiles
    (r"k_cache_attentionIfLi8ELi1ELb0E", 127),     # 256 elements
    (r"k_cache_attentionIDF16_Li8ELi1ELb0E", 62),
    (r"k_cache_attentionIDF16bLi8ELi1ELb0E", 29),
    (r"k_cache_attentionI(f|DF16_|DF16b)Li[236]ELi[12]ELb0E", 0),
    (r"k_cache_attentionI(f|DF16_|DF16b)Li4ELi1ELb0E", 0),
    (r"k_cache_attentionI(DF16_|DF16b)Li4ELi2ELb0E", 0),
])
def test_kernels_of_wide_heads_spill_no_more_registers(spills, kernel, most):  # noqa: F811
    forms = {n: s for n, s in spills.items() if re.search(kernel, n)}
    assert forms and max(forms.values()) <= most, forms
