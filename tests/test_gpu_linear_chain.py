"""Two layers with a skip connection over the second, as the header says to chain them,
against central differences in 64 bits: what the residual of the input's gradient means.

  pre = x W1^T + b1,  h = act(pre),  y = h W2^T + b2 + skip,  skip = pre or h

The gradients of x, W1 and b1 follow from dpre, the gradient of pre, which is rounded to
bf16 once (2^-8 of it; every fp32 step in front is 2^-20 of its terms at most)."""
import pytest

from helpers import stream, torch
from linear_cases import Matrix, close, lin, output, scratch_for, sync

pytestmark = pytest.mark.gpu


def check_chain(q38m, m, k, n, act, behind):
    """k inputs, n in the middle and out; behind: the skip leaves behind the activation, from h."""
    t = torch()
    call = q38m.call
    x, dy = Matrix(q38m, 1, m, k), Matrix(q38m, 2, m, n)
    w1, w2 = Matrix(q38m, 3, n, k, sigma=k ** -0.5), Matrix(q38m, 4, n, n, sigma=n ** -0.5)
    b1, b2 = Matrix(q38m, 5, 1, n, "f32"), Matrix(q38m, 6, 1, n, "f32")
    pre, h, y = output(q38m, m, n, "f32"), output(q38m, m, n), output(q38m, m, n, "f32")
    one, two = scratch_for(q38m, m, n, k)[0:3], scratch_for(q38m, m, n, n)[0:3]
    call("q38m_linear_v1", x.arg, w1.arg, b1.arg, q38m.ACTIVATIONS[act], None, h.arg, pre.arg, *one[1:], stream(), 0)
    call("q38m_linear_v1", h.arg, w2.arg, b2.arg, 0, (h if behind else pre).arg, y.arg, None, *two[1:], stream(), 0)
    dpre = output(q38m, m, n)
    if behind:  # the whole gradient of h goes through the activation
        dh = output(q38m, m, n, "f32")
        call("q38m_linear_backward_input_v1", dy.arg, w2.arg, None, 0, dy.arg, dh.arg, *two[1:], stream(), 0)
        call("q38m_linear_backward_activation_v1", dh.arg, pre.arg, q38m.ACTIVATIONS[act], dpre.arg, stream(), 0)
    else:
        call("q38m_linear_backward_input_v1", dy.arg, w2.arg, pre.arg, q38m.ACTIVATIONS[act], dy.arg, dpre.arg, *two[1:],
             stream(), 0)
    dx, dw, db = output(q38m, m, k, "f32"), output(q38m, n, k, "f32"), output(q38m, 1, n, "f32")
    call("q38m_linear_backward_input_v1", dpre.arg, w1.arg, None, 0, None, dx.arg, *one[1:], stream(), 0)
    call("q38m_linear_backward_weight_v1", dpre.arg, x.arg, None, dw.arg, db.arg, *one[1:], stream(), 0)
    sync()

    def value(x_, w_, b_):
        z = x_ @ w_.T + b_
        a = lin.activation(act, z)
        return (dy.values * (a @ w2.values.T + (a if behind else z))).sum()

    # of every term of dpre, with the activation's slope at 1.13 at most
    back = 1.13 * (dy.values.abs() @ w2.values.abs() + dy.values.abs())
    sizes = {"x": back @ w1.values.abs(), "w": back.T @ x.values.abs(), "b": back.sum(0, keepdim=True)}
    step = 2.0 ** -12
    given = {"x": x.values, "w": w1.values, "b": b1.values}
    for name, got in (("x", dx.got()), ("w", dw.got()), ("b", db.got())):
        want = t.empty(got.numel(), dtype=t.float64, device="cuda")
        for i in range(got.numel()):
            def moved(by):
                v = {key: p.clone() for key, p in given.items()}
                v[name].view(-1)[i] += by
                return value(v["x"], v["w"], v["b"])
            want[i] = (moved(step) - moved(-step)) / (2 * step)
        # the differences are off by a sixth of step^2 times a third derivative: of an activation at most
        # 4, times the third power of what the step is multiplied by
        power = {"x": w1.values.abs().max(), "w": x.values.abs().max(), "b": 1.0}[name]
        third = step * step * (1 + power ** 3) * sizes[name].max()
        close(got, want.view_as(got), sizes[name] * (2.0 ** -8 + 2.0 ** -20) + third, "f32", (name, act, behind))


@pytest.mark.parametrize("behind", [False, True])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "sigmoid"])
def test_two_layers_with_a_skip(q38m, act, behind):
    check_chain(q38m, 5, 12, 8, act, behind)
    check_chain(q38m, 3, 7, 11, act, behind)  # rows that do not start at 16 bytes
