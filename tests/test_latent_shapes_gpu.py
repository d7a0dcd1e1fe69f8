"""Shapes of the latent-cache calls at which the work is laid out otherwise than in test_latent_gpu.py, whose bounds
hold here too: appends whose waves take several groups of 16 query heads of a row, and prompts with rows in
sequences past the first 64 and the first 576 of the call."""
import numpy as np
import pytest

import test_latent_gpu as t

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,heads", [(3100, 33),   # all three groups a wave, the last of one head
                                        (2500, 70),   # four of five groups, then one
                                        (1600, 128),  # four of eight
                                        (4093, 20)])  # both
def test_append_of_several_groups_a_wave(mx, rows, heads, f8):
    groups = -(-heads // 16)
    assert rows * groups // (12 * 256) > 1  # what a wave takes
    t.test_append(mx, 512, 64, heads, 2, 64, rows, f8)


def counts(sequences, rng, live):
    """New and total positions of each sequence: some for the live ones, none (but perhaps positions) for others."""
    new, total = np.zeros(sequences, int), np.zeros(sequences, int)
    for s, (n, prior) in live.items():
        new[s], total[s] = n, n + prior
    idle = new == 0
    total[idle] = rng.integers(0, 3, idle.sum())
    return new, total


def run(mx, seed, heads, nope, new, total):
    starts, kv_starts = np.cumsum([2, *new]), np.cumsum([1, *total])
    args = t.formed(np.random.default_rng(seed), starts[-1] + 3, kv_starts[-1] + 2, heads, nope)
    got = t.run_prefill(mx, *args, starts, kv_starts, heads, nope)
    t.check_prefill(got, *args, starts, kv_starts, heads, nope)
    assert (t.run_prefill(mx, *args, starts, kv_starts, heads, nope) == got).all()


@pytest.mark.parametrize("heads,nope", [(1, 128), (3, 64), (9, 128)])
@pytest.mark.parametrize("sequences", [65, 70, 128, 600, 1100])
def test_prompts_of_many_sequences(mx, sequences, heads, nope):
    """Every sequence has rows, most a few and some more than a workgroup's 256."""
    t.say("many prompts", sequences, heads, nope)
    rng = np.random.default_rng(60 + sequences)
    live = {s: (int(rng.integers(1, 9)), int(rng.integers(0, 40))) for s in range(sequences)}
    for s in (0, 62, 63, 64, sequences - 1):
        live[s] = (257 + s % 50, s)
    run(mx, 61, heads, nope, *counts(sequences, rng, live))


@pytest.mark.parametrize("heads,nope", [(1, 128), (3, 64), (8, 128)])
@pytest.mark.parametrize("sequences,live", [
    (65, [0, 63, 64]), (70, [64, 69]), (128, [1, 127]), (600, [0, 63, 64, 65, 300, 575, 576, 599]), (600, [576]),
    (700, [575, 640, 699]), (1200, [30, 1088, 1199])])
def test_split_prompts_among_idle_sequences(mx, sequences, live, heads, nope):
    """Few rows in sequences far into the call, on prefixes long enough that the keys are split and joined."""
    t.say("split among idle", sequences, live, heads, nope)
    rng = np.random.default_rng(62)
    run(mx, 63, heads, nope, *counts(sequences, rng, {s: (int(rng.integers(1, 60)), 900 + s % 7) for s in live}))
