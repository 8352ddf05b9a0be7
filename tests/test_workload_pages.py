"""The pages of the measured step over the 4-bit cache: what the plan gives a sequence is no other sequence's."""
from types import SimpleNamespace

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import serving_reference as served
from loken_amd import workloads


@pytest.mark.parametrize("seqs,context,drafts", [(1, 1, 0), (5, 64, 0), (4, 128, 3), (3, 100, 2), (2, 63, 1), (2, 60, 64), (3, 64, 200)])
def test_sequences_share_no_page(seqs, context, drafts):
    mk = SimpleNamespace(dev="cpu", gen=torch.Generator().manual_seed(1))
    between = workloads.BetweenMxfp4(seqs * (drafts + 1), context, 8, 2, mk, drafts)
    before = between.table.numpy().copy()
    table, lens, *_, taken = served.plan(between.past.numpy(), between.fresh.numpy(), before, between.free.numpy(), workloads.PAGE_TOKENS, between.rows, 0)
    of_each = -(-(context + drafts + 1) // workloads.PAGE_TOKENS)
    used = np.asarray(table)[:, :of_each].reshape(-1)
    assert taken <= between.free.numel() and (lens == context + drafts + 1).all()
    assert ((used >= 0) & (used < between.pages)).all() and len(set(used.tolist())) == used.size
