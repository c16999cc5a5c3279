"""More calls of the paged-cache operators: every wait's last phase, and what the
descriptions of the entry points say about odd calls."""
import pytest

import paged_util as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,tile", [(128, 80), (64, 96)])
@pytest.mark.parametrize("tiles", [1, 2, 3, 4, 5, 6, 11])
def test_attention_ends_after_any_number_of_tiles(dim, tile, tiles):
    """About one item per SM: its tiles fill the ring in part, just, or several times, and every copy is waited for
    (a wait for a phase that never comes would set the timeout bit)."""
    b = P.Batch([(tile * tiles - 20, 17)] * 148, 1, 1, dim, 16, "bf16")
    b.call()
    b.check()
    assert P.device_error() == 0
