"""Verification of drafted tokens where the numbers are at the ends of their
range, or outside it, and the tokens at the ends of the rows that are drawn from
have no probability: a token with one follows all the same."""
import numpy as np
import pytest

from test_gpu_verify import VerifyCase, note

pytestmark = pytest.mark.gpu

ENDS = [0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan")]


@pytest.mark.parametrize("vocab,first,last", [(500, 3, 498), (9000, 4099, 8100), (300, 7, 8)])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("kind", ["one row", "drafts stand", "refused"])
@pytest.mark.parametrize("u", ENDS)
def test_rows_masked_at_their_ends(hip, u, kind, weights, vocab, first, last):
    note("u = %r, %s, weights=%s, vocabulary %d" % (u, kind, weights, vocab))
    lens = {"one row": [1, 1], "drafts stand": [3, 2], "refused": [3, 2]}[kind]
    starts = np.concatenate([[0], np.cumsum(lens)])
    none = 0.0 if weights else -np.inf

    def edit(t, d, tokens, uu):
        t[:, :first] = none
        t[:, last:] = none
        for s, e in zip(starts, starts[1:]):
            uu[e - 1] = u
            for r in range(s, e - 1):
                tokens[r] = first + 1 if kind == "drafts stand" else 0
                if kind == "drafts stand":  # the only token of its row: stands for any u below 1
                    t[r] = none
                    t[r, first + 1] = 1.0

    c = VerifyCase("f32", vocab, lens, "none", weights, 1.0, seed=2, edit=edit)
    accepted, nxt, _, _ = c.answer
    assert accepted == ([n - 1 for n in lens] if kind == "drafts stand" else [0] * len(lens))
    assert all(first <= v < last for v in nxt), nxt
    if not (0.0 <= u < 1.0):
        assert all(v == (first if u < 0.0 else last - 1) for v in nxt), nxt
    if u == 0.0:
        assert all(v == first for v in nxt), nxt
    c.check(hip, "ends")


@pytest.mark.parametrize("u", ENDS)
def test_what_the_draft_leaves_is_masked_at_its_ends(hip, u):
    """A refused draft whose row is the target's but for three tokens in the
    middle: what is left of it is zero at both ends."""
    note("u = %r, what is left" % u)

    def edit(t, d, tokens, uu):
        d[:] = t
        d[0, 200:203] = -np.inf
        d[2, 40:43] = -np.inf
        tokens[:] = 4999  # q > p there, and u of 1 refuses it
        uu[0] = uu[2] = 1.0
        uu[1] = uu[3] = u

    c = VerifyCase("f32", 5000, [2, 2], temp=1.0, seed=3, edit=edit)
    accepted, nxt, _, _ = c.answer
    assert accepted == [0, 0]
    assert 200 <= nxt[0] < 203 and 40 <= nxt[1] < 43, nxt
    c.check(hip, "left")
