"""The chain prover's forward pass takes a Linear layer with the activation or sum behind it in one
call: proofs and io commitments equal the oracle's in the forms where that could show."""
import numpy as np
import pytest

import oracle_lib as O
import zkml_b200 as Z
from helpers import int_matrix_m31, uniform_m31

pytestmark = pytest.mark.gpu


def small(r, c, i):
    return int_matrix_m31(r, c, 77 + i, bound=20)


def wide(r, c, i):
    return uniform_m31(r * c, 177 + i).reshape(r, c)


CIRCUITS = {
    # outputs of the model itself: small negative reals round to the word P, as the reference leaves them
    "ends in silu": lambda d: [("linear", small(d, d, 1)), ("activation", "silu")],
    "ends in gelu": lambda d: [("linear", small(d, d, 2)), ("activation", "gelu")],
    "ends in relu, wide weights": lambda d: [("linear", wide(d, d, 3)), ("relu", None)],
    "residual": lambda d: [("linear", small(d, d, 4)), ("linear", small(d, d, 5)), ("add", 0)],
    "sum of a layer with itself": lambda d: [("linear", small(d, d, 6)), ("add", 0)],
    # both the Linear output and its activation are used later
    "linear output used twice": lambda d: [("linear", small(d, d, 7)), ("relu", None), ("linear", small(d, d, 8)),
                                           ("add", 0)],
    "activation added to what follows": lambda d: [("linear", small(d, d, 9)), ("linear", small(d, d, 10), -1),
                                                   ("add", 0)],
}


@pytest.mark.parametrize("name", list(CIRCUITS))
@pytest.mark.parametrize("m,d", [(1, 16), (5, 24), (40, 64)])
def test_chain_equals_oracle(name, m, d):
    x = int_matrix_m31(m, d, m + d, bound=50)
    layers = CIRCUITS[name](d)
    rc, raw, dig, io = O.prove_gkr_chain(x, layers, n_queries=3)
    assert rc == 0
    p = Z.prove_gkr_chain(x, layers, n_queries=3)
    assert p.raw.size == raw.size and (p.raw == raw).all()
    assert p.final_digest == dig and p.io_commitment == io


def test_bad_weight_is_refused_and_the_next_proof_is_right():
    x, w = int_matrix_m31(2, 16, 1, bound=50), small(16, 16, 1)
    bad = w.copy()
    bad[15, 15] = 0x80000000
    with pytest.raises(Z.InvalidArgument, match="2\\^31"):
        Z.prove_gkr_chain(x, [("linear", bad), ("relu", None)], n_queries=3)
    rc, raw, dig, io = O.prove_gkr_chain(x, [("linear", w), ("relu", None)], n_queries=3)
    p = Z.prove_gkr_chain(x, [("linear", w), ("relu", None)], n_queries=3)
    assert (p.raw == raw).all() and p.io_commitment == io
