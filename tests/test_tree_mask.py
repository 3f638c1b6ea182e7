"""tree_mask on parents that are none: no index leaves the rows (on a GPU that would be a device assert)."""
import pytest
import torch


@pytest.mark.parametrize("bad", [5, 6, 100, 2 ** 31 - 1, -7])
def test_parents_that_do_not_come_before_their_node(bad):
    from fp4_attn_b200.paged_cache import tree_mask
    parents = torch.tensor([[-1, 0, 0, bad, 3, 2], [bad, 0, 1, 2, 3, 4]], dtype=torch.int32)
    m = tree_mask(parents)
    none = torch.tensor([[-1, 0, 0, -1, 3, 2], [-1, 0, 1, 2, 3, 4]], dtype=torch.int32)
    assert torch.equal(m, tree_mask(none))
    assert m[0, 4].tolist() == [False, False, False, True, True, False]


def test_a_node_that_is_its_own_parent_and_a_circle():
    from fp4_attn_b200.paged_cache import tree_mask
    m = tree_mask(torch.tensor([[0, 1, 3, 2]]))
    assert m[0].tolist() == [[True, False, False, False], [False, True, False, False], [False, False, True, False],
                             [False, False, True, True]]
