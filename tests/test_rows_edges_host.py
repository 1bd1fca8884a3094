"""Row operators without a GPU, at the edges of what their calls take."""
import pytest
import torch

from test_rows_host import rows   # noqa: F401  CPU tensors let through, the library out of reach


def test_half_a_pair_of_gradients_is_refused(rows):   # noqa: F811
    x, w, g = torch.zeros(4, 8), torch.zeros(3, 8), torch.zeros(4, 3)
    for pair in ((g, None), [g, None], (None, g), (g,), (g, g, g)):
        with pytest.raises(RuntimeError, match="grad_y must be a tensor or a pair"):
            rows.linear_backward(pair, x, w)
