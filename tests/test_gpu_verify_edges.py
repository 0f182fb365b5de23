"""verify and probs where their own tests do not go: sequences that fill the last warp in part,
weights that are not probabilities, vocabularies beyond a CTA's share, rows behind the last
sequence.  The restatement is test_gpu_verify's; tokens and counts have to be equal."""
import numpy as np
import pytest
import torch

from test_gpu_verify import check_verify, i32, rows_of

from lama32_mojo_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,drafts", [(9000, [33, 0, 65, 1, 31, 700]), (33000, [513]), (70000, [1, 40])])
@pytest.mark.parametrize("certain", [False, True])
def test_sequences_of_odd_lengths_over_clusters(cuda, n, drafts, certain):
    """Rows that do not fill the warps that store them, several CTAs a sequence."""
    rng = np.random.default_rng(n)
    starts = np.concatenate([[0], np.cumsum([d + 1 for d in drafts])])
    rows = int(starts[-1])
    p = rows_of(rng, rows, n)
    last = set(starts[1:] - 1)
    body = [r for r in range(rows) if r not in last]
    q = p[body]
    ids = np.zeros(rows, np.int64)
    for r in body:
        ids[r + 1] = p[r].argmax()
    u = (rng.random(rows) * 0.9).astype(np.float32)
    for b in range(len(drafts)):  # a refused draft somewhere in each
        if drafts[b]:
            u[starts[b] + rng.integers(drafts[b])] = 1.0
    check_verify(p, None if certain else q, ids, starts, u, cuda)


@pytest.mark.parametrize("S,n", [(149, 2_700_001), (1, 40_960_000)])
def test_columns_beyond_what_one_cta_holds(cuda, S, n):
    """Many sequences get few CTAs each, but never fewer than their columns need; the most columns."""
    p = torch.zeros((S, n), device=cuda)
    at = torch.arange(S, device=cuda) * ((n - 1) // max(S - 1, 1))
    at[-1] = n - 1
    p[torch.arange(S, device=cuda), at] = 1.0
    a, t = ops.verify(p, None, i32(np.zeros(S), cuda), i32(np.arange(S + 1), cuda), torch.full((S,), 0.5, device=cuda))
    assert t.tolist() == at.tolist() and not a.any()


def test_negative_and_nan_weights_of_q(cuda):
    """A negative q counts as 0: it neither keeps a draft that p gives no weight, nor adds to the
    next token's weights.  A NaN refuses its draft and takes its index out."""
    n = 300
    p = np.full((8, n), 1.0 / 128, np.float32)
    p[:, 128:] = 0.0
    q = np.full((4, n), 1.0 / 256, np.float32)
    starts, ids, u = np.array([0, 2, 4, 6, 8]), np.zeros(8, np.int64), np.full(8, 0.5, np.float32)
    ids[1], q[0, 200] = 200, -0.5  # p is 0: refused; index 200 must not be drawn
    ids[3], q[1, 5] = 5, -3.0      # p is not 0: kept, as with q = 0
    ids[5], q[2, 7] = 7, np.nan    # refused
    ids[7], q[3, 9] = 250, -1e30   # refused; index 9 weighs p(9), no more
    a, t = ops.verify(*(torch.from_numpy(x).to(cuda) for x in (p, q)), i32(ids, cuda), i32(starts, cuda),
                      torch.from_numpy(u).to(cuda))
    # 128 weights of 1/256: index i ends i + 1 of them, the first beyond half of them is 64; 127 without
    # index 7: i > 63.5, 64; 129 with index 9 twice: i + 2 > 64.5, 63
    assert a.tolist() == [0, 1, 0, 0]
    assert t.tolist() == [64, -1, 5, 64, 64, -1, 63, -1]


def test_a_drawn_token_has_a_weight(cuda):
    """Segments of 128 columns, one each for the lanes that add them up: 1 + 2^-53 + 2^-53 is 1 in the order
    of the columns and 1 + 2^-52 in a tree, so that the empty fifth segment seems to begin beyond u times
    the whole, 1 of 2.  The exact draw is the third weight, a sequential one the fourth.  And draws that
    are none (negative, NaN) give tokens with a weight."""
    n = 4096
    p = np.zeros((3, n), np.float32)
    p[:, 0] = p[:, 5 * 128] = 1.0
    p[:, 2 * 128] = p[:, 3 * 128] = 2.0 ** -53
    a, t = ops.verify(torch.from_numpy(p).to(cuda), None, i32(np.zeros(3), cuda), i32(np.arange(4), cuda),
                      torch.tensor([0.5, -0.25, float("nan")], device=cuda))
    assert int(t[0]) in (3 * 128, 5 * 128)
    assert int(t[1]) == 0 and int(t[2]) in (0, 5 * 128)
