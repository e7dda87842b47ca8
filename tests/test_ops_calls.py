"""Calls of the transformer operators at the edges of their sizes, without a GPU."""
import pytest

from test_ops import arr, plan, tensors


def test_attention_of_no_batch_entry_with_documents(pkg):
    """No batch entry: done without a device, also where documents that the batch shares stand beside an array of none."""
    p = plan(pkg, batch=0)
    p(arr(pkg, (0, 5, 4, 64)), arr(pkg, (0, 7, 2, 64)), arr(pkg, (0, 7, 2, 64)), arr(pkg, (0, 5, 4, 64)),
      q_docs=arr(pkg, (5,), "i32"), k_docs=arr(pkg, (0, 7), "i32", ptr=0))
