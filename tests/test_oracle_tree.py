"""The tree oracle against closed forms and the causal prefill oracle."""

import numpy as np

from oracle import paged_prefill as opp
from oracle import tree as otree


def test_a_chain_is_causal():
    rng = np.random.default_rng(0)
    q, k, v = rng.normal(size=(5, 4, 8)), rng.normal(size=(9, 2, 8)), rng.normal(size=(9, 2, 8))
    sees = otree.ancestors([-1, 0, 1, 2, 3])
    o, _ = otree.tree_request(q, k, v, sees, 0.3)
    np.testing.assert_allclose(o, opp.prefill_request(q, k, v, 0.3), atol=1e-14)


def test_a_branch_is_the_sequence_without_the_others():
    rng = np.random.default_rng(1)
    q, k, v = rng.normal(size=(4, 2, 8)), rng.normal(size=(10, 2, 8)), rng.normal(size=(10, 2, 8))
    o, lse = otree.tree_request(q, k, v, otree.ancestors([-1, 0, 0, 1]), 0.5)
    keep = [0, 1, 2, 3, 4, 5, 6, 7, 9]  # node 3's ancestors are 1 and 0: not node 2
    want, want_lse = otree.tree_request(q[3:], k[keep], v[keep], np.ones((1, 1), bool), 0.5)
    np.testing.assert_allclose(o[3:], want, atol=1e-14)
    np.testing.assert_allclose(lse[3:], want_lse, atol=1e-14)


def test_equal_keys_give_the_mean_and_an_empty_row_nothing():
    v = np.arange(12.0).reshape(3, 1, 4)
    o, lse = otree.tree_request(np.ones((2, 1, 4)), np.zeros((3, 1, 4)), v, np.zeros((2, 2), bool), 1.0)
    np.testing.assert_allclose(o, np.broadcast_to(v[0], (2, 1, 4)))
    assert (lse == 0).all()
    o, lse = otree.tree_request(np.ones((2, 1, 4)), np.zeros((2, 1, 4)), v[:2], np.array([[0, 0], [1, 1]], bool), 1.0)
    assert (o[0] == 0).all() and lse[0] == -np.inf
    np.testing.assert_allclose(o[1], v[:2].mean(0))
    np.testing.assert_allclose(lse[1], np.log(2))


def test_accept_and_commit_by_hand():
    parents, tokens, picks = [-1, 0, 0, 2, 2], [9, 4, 5, 6, 7], [5, 0, 7, 0, 3]
    assert otree.accept(tokens, parents, picks, [0, 5], 4) == ([[0, 2, 4, -1]], [3], [[5, 7, 3, -1]])
    assert otree.accept(tokens, parents, picks, [0, 0, 5], 2) == ([[-1, -1], [0, 2]], [0, 2], [[-1, -1], [5, 7]])
    cache = np.arange(8.0).reshape(1, 4, 1, 2, 1, 1).repeat(2, axis=2)  # slot (page p, t) holds 2 p + t
    got = otree.commit(cache, [0, 5], [0, 4], [3, 1, 0, 2], [1], [[0, 2, 4, -1]], [3])
    # 7 tokens, 2 committed: positions 2, 4, 6 (slots 2, 0, 4) to positions 2, 3, 4 (slots 2, 3, 0)
    assert got[0, :, 0, :, 0, 0].reshape(-1).tolist() == [4, 1, 2, 0, 4, 5, 6, 7]
