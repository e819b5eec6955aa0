"""Refusals of index, mask and weight pointers that are not aligned to their elements, which the kernels could not read."""
import pytest

from ramforge_b200 import _lib, kv_cache_read, kv_cache_write, qk_norm_rope, tree_attention

from .test_verify_args import KV, NR, P, TA, refused, view


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("arg", ["positions_ptr", "q_norm_ptr", "k_norm_ptr"])
def test_norm_rope_refuses_unaligned(arg, off):
    refused(qk_norm_rope, NR, {arg: P + off}, _lib.RF_EINVAL, "4-byte aligned")


@pytest.mark.parametrize("off", [1, 2])
@pytest.mark.parametrize("arg", ["pos_ptr", "seq_ptr"])
def test_cache_calls_refuse_unaligned(arg, off):
    for fn, ptrs in ((kv_cache_write, ("k_ptr", "v_ptr")), (kv_cache_read, ("k_out_ptr", "v_out_ptr"))):
        refused(fn, {**KV, "cache": view(), **dict.fromkeys(ptrs, P)}, {arg: P + off}, _lib.RF_EINVAL, "4-byte aligned")


@pytest.mark.parametrize("off", [1, 2])
@pytest.mark.parametrize("arg", ["hist_len_ptr", "n_draft_ptr", "mask_ptr"])
def test_tree_attention_refuses_unaligned(arg, off):
    refused(tree_attention, {"cache": view(), **TA}, {arg: P + off}, _lib.RF_EINVAL, "4-byte aligned")
