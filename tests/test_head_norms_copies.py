"""CPU checks that head norms are copied, deep-copied and pickled as values: a copy
passes the addresses of its own weights."""

import copy
import pickle

import pytest
import torch

from mtplx_amd.rotary import HeadNorms, _heads, head_norms, rotary_table

CPU = torch.device("cpu")


@pytest.mark.parametrize("again", [copy.deepcopy, lambda n: pickle.loads(pickle.dumps(n)), copy.copy],
                         ids=["deepcopy", "pickle", "copy"])
@pytest.mark.parametrize("sides", [(True, True), (True, False), (False, True)])
def test_a_copy_is_one_of_its_own(again, sides):
    w = [torch.rand(8) if s else None for s in sides]
    n = head_norms(*w, eps=0.25)
    m = again({"layer": n})["layer"] if again is not copy.copy else copy.copy(n)
    t = rotary_table(8, device="cpu")
    a = _heads(t, m, None, 8, CPU)
    assert (a.axes, a.eps, m.eps) == (1, 0.25, 0.25)
    for mine, theirs, address in ((m.queries, n.queries, a.q_weight), (m.keys, n.keys, a.k_weight)):
        assert (mine is None) == (theirs is None) and address == (None if mine is None else mine.data_ptr())
        if mine is not None:
            assert torch.equal(mine, theirs) and (again is copy.copy or mine.data_ptr() != theirs.data_ptr())


def test_a_copy_of_what_calls_refuse_is_refused():
    by_hand = HeadNorms(torch.ones(8), None, 1e-6)
    with pytest.raises(TypeError):
        _heads(rotary_table(8, device="cpu"), copy.deepcopy(by_hand), None, 8, CPU)
