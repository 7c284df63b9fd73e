"""Calls at the edges of what the operators around a decode step take, without a GPU: empty batches with views of other strides or
types, and sizes at which a 32-bit index or the number of workgroups of a launch would not do (described, never read).
"""
import ctypes

import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec


@pytest.fixture(scope="module")
def lib():
    return pth_dec.load_library()


def case():
    return kvc.make_case([37, 5], [3, 1], num_q_heads=12, num_kv_heads=2, block_size=16, seed=3)


def call(fn, descs, *scalars):
    err = ctypes.create_string_buffer(256)
    rc = fn(*[ctypes.byref(d) for d in descs], *scalars, None, err, len(err))
    return rc, err.value.decode()


def describe(*ts):
    return [pth_dec.describe(t) for t in ts]


def views(c):
    return c.key_cache, c.value_cache, c.k_scale, c.v_scale


# ---- no tokens ----

@pytest.mark.parametrize("dtype,out", [
    ("fp16", lambda hq: torch.empty((0, hq, 256), dtype=torch.float16)),
    ("fp32", lambda hq: torch.empty((0, hq, 256), dtype=torch.float16)),
    ("bf16", lambda hq: torch.empty((0, hq + 1, 256), dtype=torch.bfloat16)[:, 1:]),
    ("fp32", lambda hq: torch.empty((0, hq, 512))[..., :256]),
])
def test_rotary_write_of_no_tokens_into_another_tensor(lib, dtype, out):
    c = case().cache
    x = torch.empty((0, 16, 256), dtype={"fp16": torch.float16, "fp32": torch.float32, "bf16": torch.bfloat16}[dtype])
    n = torch.zeros(0, dtype=torch.int64)
    # (the data of all empty tensors is the null pointer: that does not make query_out the query)
    assert call(lib.pth_cache_write_rotary, describe(x[:, :12], out(12), x[:, 12:14], x[:, 14:], n, torch.zeros((9, 64)), *views(c), n),
                0) == (0, "")
