"""examples/tree_decoding.py: generation with drafted trees gives the tokens of generation token by token."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "tree_decoding.py")


@pytest.mark.parametrize("steps,nodes,batch", [(40, 9, 3), (25, 2, 1), (30, 40, 6)])
def test_trees_generate_what_single_tokens_do(steps, nodes, batch):
    spec = importlib.util.spec_from_file_location("tree_decoding", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    one, trees, calls = m.run(steps=steps, nodes=nodes, batch=batch)
    assert one.shape == (batch, steps) and torch.equal(one, trees)
    assert len(set(one.flatten().tolist())) > 10  # not one token over and over
    if nodes > 2:
        assert calls < steps  # drafted tokens were accepted
