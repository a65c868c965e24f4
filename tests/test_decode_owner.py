"""The split decode's search for the CTA that owns a page-group (localstack_b200/csrc/decode.cuh, cta_of), on CPU:
its first guess ceil((x + 1) G / P) - 1, in doubles as in the kernel, already is the owner for every allowed
size (G <= 512 CTAs, P below 2^31 page-groups), more CTAs than page-groups included, so the corrections that
follow it never step over empty ranges."""
import math
import os
import re

import numpy as np

K_MAX_CTAS = 512


def first_guess(x, P, G):
    return math.ceil(float(x + 1) * float(G) / float(P)) - 1


def owner(x, P, G):
    """The c with floor(c P / G) <= x < floor((c + 1) P / G), in whole numbers."""
    return ((x + 1) * G + P - 1) // P - 1


def _check(x, P, G):
    c = owner(x, P, G)
    assert 0 <= c < G and c * P // G <= x < (c + 1) * P // G
    assert first_guess(x, P, G) == c, (x, P, G)


def test_every_small_case():
    for G in list(range(1, 40)) + [74, 147, 148, 149, 255, 296, 511, 512]:
        for P in list(range(1, 60)) + [G, G + 1, 2 * G - 1, 2 * G, 3 * G + 1]:
            for x in range(P):
                _check(x, P, G)


def test_random_and_edge_cases():
    rng = np.random.default_rng(0)
    for _ in range(100000):
        G = int(rng.integers(1, K_MAX_CTAS + 1))
        P = int(2 ** rng.uniform(0, 31))
        x = int(rng.integers(0, P))
        c = int(rng.integers(0, G + 1))
        for y in (x, 0, P - 1, c * P // G, c * P // G - 1):  # the last ones: either side of a range's bound
            if 0 <= y < P:
                _check(y, P, G)


def test_the_kernel_has_this_formula():
    src = open(os.path.join(os.path.dirname(__file__), "..", "localstack_b200", "csrc", "decode.cuh")).read()
    body = re.search(r"int cta_of\(int64_t x, int64_t P, int G\) \{(.*?)\n\}", src, re.S).group(1)
    assert "int c = (int) ceil((double) (x + 1) * (double) G / (double) P) - 1;" in body
