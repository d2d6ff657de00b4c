"""The operators of training with a large vocabulary at the ends of their ranges,
against the float64 forms (oracle.vocab)."""
import numpy as np
import pytest
from devarrays import T as dev_array, empty, full
from test_vocab_gpu import host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,at", [((1 << 32) + 8, 0), ((1 << 31) + 1, 1)])
def test_dropout_of_one_row_longer_than_32_bits(dev, n, at):
    """The begin, the borders and the end of one row of n values are those of short
    calls that start there; `at` values into memory the row is taken value by value."""
    from minitorch_amd import kernels as K

    x = full((1, n + at), 1.0, "bfloat16")[:, at:]
    y = K.dropout(x, 0.5, 3, 11, out=x).view(n)
    for e in (0, (1 << 31) - 64, n // 2 // 4 * 4, n // 4 * 4 - 64):
        some = min(64, n - e)
        part = K.dropout(full((1, some), 1.0, "bfloat16"), 0.5, 3, 11 + e // 4)
        assert np.array_equal(host(y[e:e + some]), host(part)[0])
    # nothing is left as it was: every value is 0 or 2, the tail too
    assert set(np.unique(host(y[n - 8:]))) <= {0.0, 2.0}


def test_dropout_function_of_more_than_32_bits_of_values(dev):
    """F.dropout, which takes its tensor as one row, and its backward."""
    from minitorch_amd import F, Tensor
    from minitorch_amd import device as D
    from minitorch_amd import kernels as K

    n = (1 << 32) + 8
    x = Tensor(D.full((n,), 1.0), requires_grad=True)
    F.set_dropout_seed(9)
    y = F.dropout(x, 0.5)
    y.grad = D.full((n,), 3.0)
    y._backward()
    for e in (0, 1 << 31, n - 64):
        part = host(K.dropout(full((1, 64), 1.0), 0.5, 9, e // 4, subsequence=1))[0]
        assert np.array_equal(host(y.data.t[e:e + 64]), part)
        assert np.array_equal(host(x.grad.t[e:e + 64]), 3 * part)
