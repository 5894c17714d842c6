"""GPU: the launches of linear attention with a decay that need many sequences,
long ones or absent results: walks of many chunks without segments, a backward
without the rates' gradient, forwards in twice as many segments.  Tolerances are
DecayCase.tol()'s."""
import pytest
import torch

from decayref import D, DecayCase
from test_gpu_decay import NAMES, check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(n=70, t=200, h=8, hkv=8, dk=16, dv=16, reverse=3),
                                dict(n=65, t=193, h=8, hkv=4, dk=24, dv=8,
                                     lens=[193, 96, 1, 160, 0] * 13)])
def test_many_sequences_walk_whole(rnn, kw):
    """More walks than the device has places for: no segments, seven chunks each."""
    cs = DecayCase(seed=21, **kw)
    core = rnn.DecayCore(cs.h, cs.dk, cs.dv, cs.hkv)
    layout = (cs.qstride, 0, cs.kvstride, cs.koff, None, cs.voff)
    assert core._plan(cs.n, cs.t, 0, layout)[1] == 0  # a segment's state is workspace
    got, want = run(rnn, cs), cs.want()
    check(cs, got, want, cs.sizes())
    if cs.lens is not None:
        for b, m in enumerate(cs.lens.tolist()):
            assert all((got[nm][b, m:] == 0).all() for nm in ("y", "dq", "dk", "dv"))
