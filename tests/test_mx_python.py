"""Refusals of the Python conveniences of the microscaled rows, by their messages."""
import pytest
import torch


def test_rounded_values_over_the_rows(q38m):
    """Outputs overlap no input: not x itself, nor a part of its memory."""
    x = torch.zeros(6, 64, dtype=torch.bfloat16)
    both = torch.zeros(12, 64, dtype=torch.bfloat16)
    for rows, rounded in ((x, x), (x[:3], x[:3]), (both[:6], both[5:11]), (both[:, :32], both.view(-1)[300:684].view(12, 32)),
                          (both[:2, :8], both[1, 4:20].view(2, 8)), (both[5:6], both[5:6])):
        with pytest.raises(q38m.InvalidArgument, match="overlap"):
            q38m.mx_quantize(rows, rounded=rounded)
    for rows, rounded in ((x, torch.zeros_like(x)), (both[:6], both[6:]), (both[6:], both[:6]), (x, None),
                          (both[:2, :8], both[1, 8:24].view(2, 8)), (both[:2, :8], both[0, 48:].view(2, 8)),
                          (both[:2, :8], both[0, 8:24].view(2, 8))):
        with pytest.raises(q38m.InvalidArgument, match="on a GPU"):  # the next check
            q38m.mx_quantize(rows, rounded=rounded)
