"""A call that fails says so once: the calls behind it, on the same index or another one, start clean."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _answers(ix, rows):
    scores, ids = ix.query(rows[2], 3)
    return ids[0] == 2 and np.isfinite(scores).all()


def test_an_allocation_that_is_refused_leaves_no_error_for_the_next_call():
    import torch

    from morphik_core_amd import MvError
    from morphik_core_amd.index import MvIndex, synth_rows

    rows = [synth_rows(5, i, 32) for i in range(8)]
    ix = MvIndex(capacity_pages=8, stride_rows=32)
    ix.add(rows)
    assert _answers(ix, rows)
    _free, total = torch.cuda.mem_get_info(0)
    for kw in (dict(), dict(with_fde=True), dict(with_float=False, with_fp8=True)):
        with pytest.raises(MvError, match="hipMalloc|memory"):
            MvIndex(capacity_pages=int(2 * total // (1024 * 128)), stride_rows=1024, **kw)  # one slab of at least twice the card
        other = MvIndex(capacity_pages=4, stride_rows=32, with_fde=True)  # its tables end with a check of the last error
        other.add(rows[:4])
        assert _answers(other, rows) and _answers(ix, rows)
        other.close()
    ix.close()
