"""Calls of the paged cache beside one another: plans of one kernel instance with different shared memory, captured steps
that reuse their buffers, other streams, and what a bad value or a failed call leaves behind."""
import numpy as np
import pytest

import backburner_b200 as pa
from backburner_b200 import api
from test_cache_gpu import Seqs, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant,first,second", [(pa.F16, (8, 1), (8, 64)), (pa.Q8_0, (8, 1), (2, 1)), (pa.Q4_0, (8, 3), (2, 70))])
def test_plans_of_one_kernel_keep_their_shared_memory(ctx, quant, first, second):
    """two live plans of one split-K instance, the larger one made first: neither takes the other's launch away"""
    made = []
    ctx.set_kernel(1)
    for nkv, tok in (first, second):
        sq = Seqs(nkv + tok, [200, 77], 128, nkv, quant)
        made.append((sq, tok, pa.CachePlan(ctx, sq.cache, 2, tok, 1, sq.max_pages)))
    ctx.set_kernel(0)
    for i in (0, 1, 0, 1):
        sq, tok, plan = made[i]
        Qs = sq.q(tok, 1)
        out = plan.reply(sq.layer, Qs, sq.table, sq.n_keys)
        ctx.status()
        _check(sq, Qs, out, tok, 1)
    for _, _, plan in made:
        plan.close()
