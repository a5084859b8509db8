"""Attention weights of a shard, hand-worked: which of its tokens are new goes by the whole sequence."""

import numpy as np
import pytest

from oracle import weights_reference


@pytest.mark.parametrize("held,mask,new", [(8, 8, 2), (8, 20, 0), (8, 9, 1), (2, 2, 2), (1, 2, 1), (8, 6, 4)])
def test_new_tokens_of_a_shard(held, mask, new):
    """q_len 2, equal scores and lse 0: a row's weight of every token it sees is 1, old scores are 10.
    Row qi sees t < mask - 1 + qi; tokens from mask - 2 on are new."""
    q, kc = np.zeros((1, 2, 4, 128)), np.zeros((1, 16, 1, 128))
    scores, _ = weights_reference(q, kc, np.ones((1, 1)), np.array([[0]]), [held], np.zeros((1, 2, 4)), np.full((1, 1, 16), 10.0),
                                  mask_lens=[mask])
    want = [4.0 * ((t < mask - 1) + (t < mask)) + (10.0 if t < mask - 2 else 0.0) for t in range(held)]
    assert scores[0, 0, :held].tolist() == want and (scores[0, 0, held:] == 10).all()
    assert sum(w < 10 for w in want) == new
