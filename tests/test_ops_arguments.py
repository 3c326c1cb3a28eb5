"""Arguments of the operators of include/quantpack_ops.h that are looked at on the host, without a kernel running."""
import pytest
import torch

from test_ops_refusals import lib, weight_args  # noqa: F401  (the fixture)


def test_key_weights_of_sequences_without_pages(lib):  # noqa: F811
    """A block table of no columns holds no position: there is nothing to do, whether it has an address or not."""
    assert lib.qp_key_weights(weight_args(max_blocks=0), None) == 0
    assert lib.qp_key_weights(weight_args(max_blocks=0, block_table=None), None) == 0
