"""GPU tests of the verification of drafts (tlg_dev_spec_verify) where its launches
change: a workgroup a sequence, or two launches over all rows."""
import pytest

from test_serve_gpu import BF16, F16, F32, Drafts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("rows,V", [
    ([8], 2048), ([9], 2048), ([16], 131), ([17], 131), ([400], 33), ([200, 1, 0, 3], 1001), ([1] * 256, 40), ([1] * 257, 40),
    ([64] + [1] * 127, 50), ([4200] + [1] * 127, 17), ([3, 2] * 64, 4100)])
def test_verify_at_the_launches_borders(lib, type, drafted, rows, V):
    d = Drafts(rows, V, type, drafted, seed=V + len(rows), pad=3, lead=1, tail=2, scale=0.9, dscale=1.1, agree=0.2)
    d.check(d.run(lib))
