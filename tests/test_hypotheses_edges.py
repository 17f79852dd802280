"""Several hypotheses of a request on the host: limits that the operators name, books that stay whole, refusals of the searches and of the
command line."""

import pytest
import torch

from layover_b200 import ops

I32 = torch.int32


# ------------------------------------------------------------------------------- limits
@pytest.mark.parametrize("requests, beams, vocab", [(1, 1, 2 ** 31 - 3600), (1, 1, 2 ** 31 - 2 ** 15 + 1), (1, 64, 2 ** 25), (2, 3, 2 ** 30)])
def test_beam_selection_names_its_largest_sizes(requests, beams, vocab):
    """Places of beams x vocabulary, and the ends of the pieces that are read ahead, are counted in 32 bits."""
    f = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="meta")
    with pytest.raises(ValueError, match="at most"):
        ops.beam_select(f(requests * beams, vocab), f(requests, beams), f(requests, 4), f(requests, 4, dtype=I32), f(requests, 4, dtype=I32))


@pytest.mark.parametrize("call, message", [
    (lambda m: ops.copy_pages(m(2, 3, 4), m(65_536, dtype=I32), m(65_536, dtype=I32)), "at most 65535"),
    (lambda m: ops.copy_pages(m(65_536, 3, 4), m(1, dtype=I32), m(1, dtype=I32)), "at most 65535"),
    (lambda m: ops.compact_tokens(m(2, 3, 1, 4, 4), m(65_536, 2, dtype=I32), m(65_536, dtype=I32), m(5, dtype=I32), m(65_537, dtype=I32)), "at most 65535"),
    (lambda m: ops.compact_tokens(m(2 ** 16, 1, 2 ** 10, 1, 2 ** 9), m(1, 2, dtype=I32), m(1, dtype=I32), m(5, dtype=I32), m(2, dtype=I32)), "at most"),
])
def test_moves_name_their_largest_sizes(call, message):
    with pytest.raises(ValueError, match=message):
        call(lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="meta"))
