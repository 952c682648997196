"""The 64-bit forms that the attention kernels are held to, against central differences of their own
forward pass (on the CPU)."""
import pytest
import torch

from _attention_ref import window_attention


@pytest.mark.parametrize("q_len,kv_len,window,sinks,lengths,first", [
    (7, 7, 3, 0, None, None), (9, 9, 4, 2, [9, 5], None), (4, 12, 5, 1, [12, 6], [7, 2]),
    (5, 6, 100, 0, None, [-2, 1]), (3, 10, 2, 3, [0, 10], [4, 6])])
def test_window_attention_gradients_match_differences(q_len, kv_len, window, sinks, lengths, first):
    """Step 1e-5: its square times third derivatives of order 10 is 1e-9, rounding of a sum of order 100
    over the step 1e-9; 1e-7 is allowed."""
    g = torch.Generator()
    g.manual_seed(q_len * 31 + kv_len)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x = [r(2, q_len, 4, 6), r(2, kv_len, 2, 6), r(2, kv_len, 2, 6)]
    dout = r(2, q_len, 4, 6)
    f = lambda x: float((window_attention(*x, window, sinks, 0.4, lengths, first)[0]["out"] * dout).sum())  # noqa: E731
    got, _ = window_attention(*x, window, sinks, 0.4, lengths, first, dout)
    for at, name in enumerate(("dq", "dk", "dv")):
        for _ in range(3):
            v = r(*x[at].shape)
            up, down = ([y + s * 1e-5 * v if i == at else y for i, y in enumerate(x)] for s in (1, -1))
            assert abs((f(up) - f(down)) / 2e-5 - float((got[name] * v).sum())) <= 1e-7, name
