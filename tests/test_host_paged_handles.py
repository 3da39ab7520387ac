"""The paged cache's handles hold their tensors' addresses, taken when they are made: a field cannot be set to another tensor, which
the calls would not see. No GPU."""
import pytest

import util  # noqa: F401  (puts the package on the path)
import fv_sdpa


@pytest.mark.parametrize("cls,names", [(fv_sdpa.PagedKv, ("k", "v", "k_scales", "v_scales", "d", "kv_heads", "page_tokens", "four_bits")),
                                       (fv_sdpa.PagedBatch, ("q_start", "lens", "table"))])
def test_fields_cannot_be_set(cls, names):
    handle = cls.__new__(cls)
    for name in names:
        with pytest.raises(AttributeError):
            setattr(handle, name, None)
