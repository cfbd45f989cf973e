"""Which drafts the loop over drafted tokens accepts, without a GPU: the pass over them is played by a function from a path of tokens to what follows it."""
import itertools
from types import SimpleNamespace

import numpy as np
import pytest

from tensorlisp_b200.programs import DecoderConfig, TreeDecodeLoop

CFG = DecoderConfig(n_layers=1, d_model=64, n_heads=1, n_kv_heads=1, head_dim=64, d_ffn=64, vocab=100)


class Pass:
    """Takes the inputs of a step and answers for every row with the token that follows the path from the root to it."""

    def __init__(self, follows):
        self.follows, self.inputs = follows, {}

    def set_input(self, i, a):
        self.inputs[i] = np.array(a)

    def run(self):
        pass

    def read(self, _):
        ids, parents = self.inputs["ids"], self.inputs["parents"]
        out = np.zeros(ids.shape, np.float32)
        for b, i in itertools.product(*map(range, ids.shape)):
            path, at = [], i
            while at >= 0:
                path.insert(0, int(ids[b, at]))
                at = parents[b, at]
            out[b, i] = self.follows(path)
        return out


def loop(batch, drafts, follows):
    x = TreeDecodeLoop.__new__(TreeDecodeLoop)
    x.batch, x.drafts, x.max_ctx, x.cfg, x.steps = batch, drafts, 64, CFG, 0
    x.tables = np.arange(batch * 4, dtype=np.int32).reshape(batch, 4)
    x.due, x.context = np.full(batch, 7, np.int32), np.zeros(batch, np.int32)
    x.dg = SimpleNamespace(inputs={n: n for n in "ids pos tables context counts parents slots targets".split()}, token="token")
    x.prog, x.kept = Pass(follows), []
    x._keep = lambda path, kept: x.kept.append((path.copy(), kept.copy()))
    return x


@pytest.mark.parametrize("drafted,gained,path", [
    ([], [8], [0]), ([(8, -1)], [8, 9], [0, 1]), ([(5, -1)], [8], [0]), ([(8, -1), (9, 0), (5, 1)], [8, 9, 10], [0, 1, 2]),
    ([(5, -1), (8, -1), (6, 0), (9, 1)], [8, 9, 10], [0, 2, 4]),
    # the same token twice: the copy whose path goes on
    ([(8, -1), (8, -1), (9, 1)], [8, 9, 10], [0, 2, 3]), ([(8, -1), (8, -1), (9, 1), (9, 0), (10, 3)], [8, 9, 10, 11], [0, 1, 4, 5]),
    ([(8, -1), (9, 0), (9, 0), (10, 2), (8, -1), (9, 4), (10, 5), (11, 6)], [8, 9, 10, 11, 12], [0, 5, 6, 7, 8]),
    ([(8, -1), (8, -1)], [8, 9], [0, 1]), ([(5, -1), (9, 0), (8, -1)], [8, 9], [0, 3])])
def test_the_longest_path_that_agrees(drafted, gained, path):
    x = loop(2, 12, lambda p: p[-1] + 1)
    out = x.step([drafted, []])
    assert out == [gained, [8]]
    got, kept = x.kept[0]
    assert kept.tolist() == [len(path), 1] and got[0, :len(path)].tolist() == path
    assert x.context.tolist() == [len(path), 1] and x.due.tolist() == [gained[-1], 8]


def test_random_trees():
    """Against the definition: of all nodes whose path from the root agrees, one of the deepest."""
    rng = np.random.default_rng(3)
    for _ in range(300):
        n = int(rng.integers(0, 12))
        drafted = [(int(rng.integers(8, 11)), int(rng.integers(-1, i))) for i in range(n)]
        x = loop(1, 12, lambda p: 8 + sum(p) % 3)
        new = x.step([drafted])[0]
        paths, best = [[7]], [7]
        for token, parent in drafted:
            paths.append(paths[parent + 1] + [token])
            if all(paths[-1][j] == 8 + sum(paths[-1][:j]) % 3 for j in range(1, len(paths[-1]))) and len(paths[-1]) > len(best):
                best = paths[-1]
        assert new == best[1:] + [8 + sum(best) % 3]
        got, kept = x.kept[0]
        at = got[0, :kept[0]].tolist()
        assert at == sorted(set(at)) and [([7] + [t for t, _ in drafted])[i] for i in at] == best and all(drafted[b - 1][1] + 1 == a for a, b in zip(at, at[1:]))
