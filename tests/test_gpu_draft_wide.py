"""Steps with drafted tokens in 16 bits and of many columns, where the attention
runs on tensor memory, by the forms and tolerances of test_gpu_draft.py."""
import pytest
import torch

from distcomp_b200 import engine
from test_gpu_draft import TYPES, _quiet, make, tree_check  # noqa: F401
from test_gpu_kv4 import filled, rows

pytestmark = pytest.mark.gpu

WIDE = [(hd, dtype) for hd in (64, 128) for dtype in TYPES[1:]]
KV, REP = 8, 8


@pytest.mark.parametrize("hd,dtype", WIDE)
def test_a_build_with_other_registers(hd, dtype):
    """Where the kernel on tensor memory was compiled to other registers than its roles share, the other one takes the
    call; the next one is on tensor memory again."""
    lens, new = [700, 200, 1000, 64] * 3, [16, 24, 9, 40] * 3
    pool, vals = filled(KV, hd, lens, 3)
    masks, mask = make(8, new)
    q = rows(5, sum(new), KV * REP, hd).to(dtype)
    engine.inject_tree_registers()
    got = pool.attend_tree(0, q, range(12), new, mask)
    tree_check(pool, vals, q, range(12), new, masks, got, every=13)
    again = pool.attend_tree(0, q, range(12), new, mask)
    tree_check(pool, vals, q, range(12), new, masks, again, every=13)
    assert not torch.equal(got, again)
    with pytest.raises(engine.EngineError):
        engine.inject_tree_registers(-1)
