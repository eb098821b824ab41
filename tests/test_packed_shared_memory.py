"""Results of the layer norm that are one and the same tensor, refused like any other two that share memory, and refusals in front of
the first launch.  Host-side checks, no device needed."""
import pytest

from test_packed_refusals import ARGUMENT, UNAVAILABLE, fake, mt, refused  # noqa: F401 (fixtures)


def test_one_tensor_as_output_and_statistic(mt, fake):  # noqa: F811
    """Rows of one value: mean and ivar have the output's sizes."""
    shape = (4, 3, 5, 1)
    out, x, mean, ivar = (fake.tensor(*shape) for _ in range(4))
    gamma, beta = fake.tensor(1, 1, 1, 1), fake.tensor(1, 1, 1, 1)
    f = mt.Fused.LayerNormForward
    refused(mt, ARGUMENT, "memory", f, out, x, gamma, beta, out, ivar)
    refused(mt, ARGUMENT, "memory", f, out, x, gamma, beta, mean, out)
    refused(mt, ARGUMENT, "memory", f, out, x, gamma, beta, mean, mean)
    refused(mt, ARGUMENT, "memory", f, out, x, gamma, beta, x, ivar)
    refused(mt, ARGUMENT, "memory", f, x, x, gamma, beta, x, ivar)


@pytest.mark.parametrize("packed", [False, True])
def test_one_tensor_as_error_and_gradient(mt, fake, packed):  # noqa: F811
    """A batch of one: the gradients of gamma and beta have the error's sizes."""
    shape = (1, 3, 5, 6)
    error, dgamma, dbeta, delta, gamma = (fake.tensor(*shape) for _ in range(5))
    x, mean, ivar = fake.packed(*shape) if packed else fake.tensor(*shape), fake.tensor(1, 1, 1, 1), fake.tensor(1, 1, 1, 1)
    f = mt.Fused.LayerNormBackward
    refused(mt, ARGUMENT, "memory", f, error, error, dbeta, delta, gamma, x, mean, ivar)
    refused(mt, ARGUMENT, "memory", f, error, dgamma, error, delta, gamma, x, mean, ivar)
    refused(mt, ARGUMENT, "memory", f, error, error, None, delta, gamma, x, mean, ivar)
    refused(mt, ARGUMENT, "memory", f, delta, delta, dbeta, delta, gamma, x, mean, ivar)
    refused(mt, ARGUMENT, "memory", f, error, dgamma, dgamma, delta, gamma, x, mean, ivar)
    refused(mt, ARGUMENT, "memory", f, gamma, dgamma, dbeta, delta, gamma, x, mean, ivar)


def test_nothing_is_launched_before_a_refusal(mt):  # noqa: F811
    """More long rows than one launch takes: said before GeLU's derivative is written into the error."""
    at = [1 << 44]

    def tensor(*shape):
        at[0] += 1 << 42
        return mt.CTensor.wrap(at[0], shape)

    rows, n = 3_400_000, 20000
    for func in (None, "gelu"):
        args = [tensor(rows, 1, n, 1), tensor(1, 1, n, 1), tensor(1, 1, n, 1), tensor(rows, 1, n, 1), tensor(1, 1, n, 1), tensor(rows, 1, n, 1), tensor(rows, 1, 1, 1), tensor(rows, 1, 1, 1)]
        refused(mt, UNAVAILABLE, "too many", mt.Fused.LayerNormBackward, *args, beta=tensor(1, 1, n, 1), func=func)
