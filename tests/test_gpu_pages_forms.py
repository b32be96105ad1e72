"""Every form that the page calls launch, by numbers of rows and entries: up to 1024 rows or more, up to 65536 entries or more (pages then go back by a launch
of their own), and rows of several pieces of 1024 entries, each against the sequential model after every call."""
import numpy as np
import pytest

from pages_ref import Tables
from test_gpu_pages import Pair

pytestmark = pytest.mark.gpu


class ManyPages(Tables):
    def compact(self):
        """The moves of Tables.compact, the lowest ids made a set once."""
        refs = self.refs()
        used = [p for p in self.managed if refs[p]]
        lowest = self.managed[:len(used)]
        low = set(lowest)
        to = dict(zip([p for p in used if p not in low], [p for p in lowest if not refs[p]]))
        self.rows = [[to.get(p, p) for p in row] for row in self.rows]
        return list(to.items())


def pair(R, M, N):
    p = Pair(R, M, N, layers=1, kv_heads=1)
    p.model = ManyPages(p.model.rows, p.model.lens, p.model.managed, N, 16, M)
    return p


def wants(rng, lens, most):
    """Rows that grow, keep, end, get shorter by a little or by a lot, and are left alone."""
    kind, lens = rng.random(len(lens)), np.array(lens)
    return np.select([kind < 0.5, kind < 0.6, kind < 0.7, kind < 0.8, kind < 0.9],
                     [np.minimum(lens + rng.integers(0, 40, len(lens)), most), 0, np.maximum(lens - 5, 0), rng.integers(0, most + 1, len(lens)), lens], -1).tolist()


def forks(rng, R, share):
    return np.where(rng.random(R) < share, rng.integers(0, R, R), -1).tolist()


# launches: one that gives back and hands out (rows in one round), a release before it; the same for rows in several rounds
@pytest.mark.parametrize("R, M, pages_a_row", [(256, 256, 40), (1000, 65, 20), (300, 300, 40), (1024, 128, 30), (1500, 40, 12), (2600, 25, 8), (1500, 70, 20), (1025, 2, 1.5)])
@pytest.mark.parametrize("seed", range(2))
def test_random_steps_of_many_rows(R, M, pages_a_row, seed):
    rng = np.random.default_rng(100 * seed + R + M)
    N, most = int(R * pages_a_row), M * 16
    p = pair(R, M, N)
    p.resize(rng.integers(0, min(most, int(28 * pages_a_row)) + 1, R).tolist())
    for _ in range(3):
        p.fork(forks(rng, R, 0.3))
        p.resize(wants(rng, p.model.lens, most))
        p.resize(wants(rng, p.model.lens, most))
        p.compact()
    p.resize([0 if r % 3 else -1 for r in range(R)])
    p.resize([most] * R)                  # more than there are: the first rows are served
    p.resize([0] * R)


@pytest.mark.parametrize("R, M", [(1500, 40), (1500, 70), (300, 300)])
def test_shared_last_pages_in_every_round(R, M):
    """Groups whose rows lie in different rounds of 1024 write on one page; in the second step some of them end instead."""
    p = pair(R, M, 4 * R)
    p.resize([20 if r < 50 else 0 for r in range(R)])
    p.fork([r % 50 for r in range(R)])
    p.resize([21 + r % 7 for r in range(R)])
    assert p.model.failed == 0
    p.fork([r - 100 if r >= 100 and r % 2 else -1 for r in range(R)])
    p.resize([0 if r % 5 == 0 else n + 1 for r, n in enumerate(p.model.lens)])
    p.resize([n + 1 if r % 4 else -1 for r, n in enumerate(p.model.lens)])


# rows of one piece and a little, of two and a half, and of four
@pytest.mark.parametrize("R, M, N", [(70, 1025, 30000), (40, 2500, 70000), (1, 4096, 4096), (9, 4096, 20000)])
def test_rows_of_several_pieces(R, M, N):
    rng = np.random.default_rng(R + M)
    p, most = pair(R, M, N), M * 16
    lens = rng.integers(most // 3, most + 1, R)
    lens[np.cumsum(-(-lens // 16)) > N * 0.8] = 0
    p.resize(lens.tolist())
    assert p.model.failed == 0
    ends = [0, 1, 1023 * 16, 1024 * 16 - 1, 1024 * 16, 1024 * 16 + 1, 1025 * 16, 2047 * 16 + 3, 2048 * 16, 2048 * 16 + 1, most - 1, most]
    for turn in range(4):
        p.resize([min(most, ends[(r + 5 * turn) % len(ends)]) if (r + turn) % 3 == 0 else -1 for r in range(R)])
        p.fork(forks(rng, R, 0.4))
        p.resize([min(most, n + 1) if (r + turn) % 2 else -1 for r, n in enumerate(p.model.lens)])
    p.compact()
    p.resize([0 if r % 2 else -1 for r in range(R)])
    p.compact()


def test_forks_that_differ_in_a_later_piece_only():
    p = pair(6, 2500, 12000)
    p.resize([1500 * 16, 0, 0, 0, 2300 * 16 + 5, 0])
    p.fork([-1, 0, 0, 0, -1, 4])                       # all pieces of the children
    p.resize([1500 * 16 + 1, 1500 * 16 + 1, 2100 * 16, 1024 * 16, -1, 2300 * 16 + 6])
    p.fork([1, 2, 3, 0, 5, 4])                         # first pieces alike: the second and the third differ, or end earlier
    p.fork([3, 3, 3, 3, 3, 5])
    p.resize([1024 * 16 + 1] * 4 + [1023 * 16, 1024 * 16 - 3])
    p.fork([-1, 4, -1, 5, -1, 0])
    p.resize([0, 1, 2, 3, 4, 5])
