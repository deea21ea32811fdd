"""CPU test of the GPU tests' own sharpness: in the inputs of kvq8_cases a single slot
that a row sees too much or too little, a mask that is ignored or a block that is
lost moves the 64-bit result past the bound that the kernels are held to."""

import random

import pytest
import torch

import kvq8_cases as K


@pytest.mark.parametrize("args", K.CASES, ids=lambda a: "-".join(map(str, a)))
def test_a_planted_mistake_passes_the_bound(args):
    c = K.case(*args, "cpu")
    see = K.visible(c)
    r = random.Random(5)
    H, T, slots = c["H"], c["T"], c["slots"]
    carries = c["carries"]

    def moves(t, changed, head):
        a = K.attention(c, c["q"], see, [t], [head])
        other = see.clone()
        other[t] = changed
        return K.wrong(K.attention(c, c["q"], other, [t], [head]), a)

    for _ in range(12):
        t, head = r.randrange(T), r.randrange(H)
        row = see[t]
        seen, unseen = (row & carries).nonzero().flatten().tolist(), (~row & carries).nonzero().flatten().tolist()
        mistakes = []
        if seen:
            mistakes += [seen[0], seen[-1], r.choice(seen)]  # a key lost: at either end of what the row sees, inside
        if unseen:
            mistakes += [r.choice(unseen)]
            mistakes += [j for j in unseen if j and bool(row[j - 1])][:2]  # one beyond a range's end or a mask bit
            mistakes += [j for j in unseen if j + 1 < slots and bool(row[j + 1])][:2]
        for j in mistakes:
            changed = row.clone()
            changed[j] = ~changed[j]
            assert moves(t, changed, head), (t, head, j)
        if seen:
            lo = r.choice(seen) // 128 * 128  # a whole key block lost
            changed = row.clone()
            changed[lo:lo + 128] = False
            assert moves(t, changed, head)
        if c["mask"] is not None and bool((K.visible({**c, "mask": None})[t] != row).any()):
            assert moves(t, K.visible({**c, "mask": None})[t], head)  # the row's mask ignored


def test_every_row_and_edge_carries_a_value():
    for args in K.CASES:
        c = K.case(*args, "cpu")
        see = K.visible(c)
        assert bool((see & c["carries"]).any(1)[see.any(1)].all())
        assert int(c["v"].float().sum()) >= 1 and c["v"].float().ne(0).sum(1).max() <= K.PER_CHANNEL + 1
