"""Drafted tokens on the GPU: calls at the edges of what they take."""
import numpy as np
import pytest

from kv4_model import Batch
from test_gpu_draft import MODES, up, verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", MODES)
def test_verification_without_rows(holo, mode):
    """Entries without rows beside others get 0 and -1 over what was there; a batch without any writes nothing."""
    print(f"case verify no rows {mode}", flush=True)
    p = np.full((3, 40), 1 / 40, np.float32)
    u = np.full(3, 0.5)
    path, n_path, after = verify(holo, [0, 2, 0, 1, 0], [[], [-1, 0], [], [-1], []], np.int32([0, 50, 0]), u, p, p, mode)
    assert n_path.tolist() == [0, 1, 0, 1, 0] and after[[0, 2, 4]].tolist() == [-1] * 3 and path.tolist() == [0, -1, 0]
    outs = [up(holo, np.full(3, x, np.int32)) for x in (5, 6, 7)]
    ins = [up(holo, x) for x in (p, np.zeros(3, np.int32), np.full(3, -1, np.int32), np.float32(u))]
    b = Batch(holo, [0, 0, 0], max_rows=4)
    assert b.desc.rows == 0
    target, tokens, parent, us = (x.ptr for x in ins)
    assert holo.lib().holo_draft_verify(*[o.ptr for o in outs], target, target, 40, 40, 40, tokens, parent, us,
                                        MODES.index(mode), b.ref) == 0
    holo.lib().cuda_sync()
    holo.check("no rows")
    assert [o.download(np.int32).tolist() for o in outs] == [[5] * 3, [6] * 3, [7] * 3]
