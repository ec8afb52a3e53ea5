"""Lengths and rates at which the tests of forgetting look: how often a state's memory the tokens are."""

import numpy as np

# tokens, and tokens times 1 - a: below one, so that what is forgotten still grows with it
KEPT = [(16, (0.3, 1.0)), (250, (0.3, 1.0)), (4096, (0.3, 1.0)), (65536, (0.7, 1.0))]
# up to several memories
CONSTANT = [(40, (1.0, 4.0)), (1000, (1.0, 4.0)), (20000, (1.0, 6.0)), (65536, (2.0, 6.0))]


def rates(S, times, n):
    return np.linspace(*times, n) / S
