"""Trees of drafted tokens whose queries hold infinities: what every spoiled row comes to, by the formula."""
import math

import pytest
import torch

from test_gpu_paged_tree import DEV, Trees, ancestors, pack, path, queries, some_tree  # noqa: F401
from VAR_Q import _cabi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kb,vb", [(8, 8), (4, 2)])
def test_rows_of_infinite_queries(dtype, value, D, kb, vb, path):  # noqa: F811
    """a key that has a positive element (by the sign of the infinity) where the query is infinite, or a zero there, makes its score infinite or no number, and the row
    NaN throughout; where every key that the row sees scores minus infinity, none has a weight: zeros, and a sum of none"""
    counts = [40, 26, 3]
    b = Trees([300, 90, 5], 2, D, kb, vb, page=16, seed=1)
    see = [ancestors(some_tree(c, c)) for c in counts]
    see[2][0] = see[2][1] = False
    see[2][0, 0] = see[2][1, 1] = True                                        # rows of few keys, whose scores may all have one sign
    tree = torch.cat([pack(s, 2) for s in see]).to(DEV)
    q = queries(69, 8, D, dtype)
    ref, ref_lse = b.attend(q, counts, D ** -0.5, tree=tree)
    spoiled = [(7, 3, 5), (41, 0, 0), (65, 7, D - 1)] + [(66 + i % 2, h, (7 * h + i) % D) for h in range(8) for i in range(2)]
    bad = torch.zeros((69, 8), dtype=torch.bool, device=DEV)
    for t, h, d in spoiled:
        bad[t, h] = True
        q[t, h, d] = value
    out, lse = b.attend(q, counts, D ** -0.5, tree=tree)
    assert torch.equal(out[~bad], ref[~bad]) and torch.equal(lse[~bad], ref_lse[~bad])
    kinds = set()
    for t, h, d in spoiled:
        s = 0 if t < 40 else 1 if t < 66 else 2
        first = (0, 40, 66)[s]
        k = b.cache.read(b.slots[s].to(DEV))[0][:, h // 4].double()
        n, c = b.kv[s], counts[s]
        seen = torch.ones(n, dtype=torch.bool)
        seen[n - c:] = see[s][t - first]
        score = (k @ q[t, h].double())[seen.to(DEV)]
        none = bool((score == -math.inf).all())
        assert none or bool((score.isnan() | (score == math.inf)).any())      # an infinite query leaves no finite score
        kinds.add(none)
        if none:
            assert (out[t, h] == 0).all() and lse[t, h] == -math.inf, (t, h)
        else:
            assert out[t, h].isnan().all() and lse[t, h].isnan(), (t, h)
    assert False in kinds
    assert _cabi.device_status() == 0
