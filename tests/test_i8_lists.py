"""Lists of ContractionI8Plan that do not have an entry for each loop."""
import pytest

import einsum_ir_amd as eir


@pytest.mark.parametrize("name", ["dim_types", "strides_left", "strides_right", "strides_out", "strides_scale_left",
                                  "strides_scale_right", "strides_bias"])
@pytest.mark.parametrize("change", [lambda v: v[:-1], lambda v: v + [0], lambda v: []])
def test_refuses_lists_of_other_lengths(name, change):
    """Refused before the library reads past a list's end."""
    good = eir.contraction_i8_loops("tk,ok->to", dict(t=4, k=8, o=6), scale_left="t", scale_right="o", bias="o")
    with pytest.raises(ValueError, match=name):
        eir.ContractionI8Plan(**dict(good, **{name: change(good[name])}))
