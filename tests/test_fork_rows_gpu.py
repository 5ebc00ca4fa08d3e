"""What stands in a row of the page table behind its end is no page of it, whatever it is."""
import pytest

from test_kv_sequences_gpu import pools, reported, run_fork

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,P", [(3, 6), (1100, 9)])
def test_entries_behind_a_rows_end_are_not_looked_at(E, P):
    """A fork of rows with pages, and numbers that are no pages, behind their first negative entry: the definition's result, and nothing to report."""
    caches = pools(1, 3 * E + 20, 1, 64, 16)
    behind = [[-1, 10 ** 6, -1, 5], [-1, 5, 2 ** 31 - 1, -1], [-7, 6, -2, 99999]]
    lengths = [(7 * e) % 32 for e in range(E)]
    table = [[2 * e, 2 * e + 1] + behind[e % 3] + [-1] * (P - 6) for e in range(E)]
    uses = [1] * (2 * E) + [0] * (E + 20)
    state = run_fork(caches, uses, table, lengths, [0] + list(range(E - 1)), 5, 16)
    run_fork(caches, *state, None, 0, 16)   # (raises if there was something)
    # an entry that is too large in front of all negative ones is one
    table[E - 1][2] = 10 ** 6
    run_fork(caches, uses, table, lengths, None, 0, 16)
    reported(caches, "page")
