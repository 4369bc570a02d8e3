"""Rows that one launch of the router cannot take: refused, on the host.  No GPU."""
import pytest
import torch

import quantised_bayesian_nets_amd as q
from quantised_bayesian_nets_amd import _lib


def test_more_rows_than_a_launch_has_threads_for():
    """64 rows a workgroup of up to 512 threads: 2^29 rows are 2^32 threads, of which a launch would lose some without an error."""
    for T in (1 << 29, (1 << 31) - 64):
        with pytest.raises(ValueError, match="too many rows"):
            q.route_experts(torch.zeros(1, 1).expand(T, 1), 1)
    with pytest.raises(RuntimeError, match="MI355X only"):
        q.route_experts(torch.zeros(1, 1).expand((1 << 29) - 1, 1), 1)


def test_the_c_entry_refuses_them():
    L = _lib.lib()
    assert L.qbnn_route_experts(_lib.ROUTE.pack(*[1 << 20] * 9, 1, 1 << 29, 1, 1, 1, 1, 0, 0, 0, 1.0), None) == -1
    assert b"rows" in L.qbnn_last_error()
