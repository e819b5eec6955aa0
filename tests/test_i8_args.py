"""Refusals of the 8-bit row calls and of the verdict on drafted tokens: wrong arguments give RF_EINVAL with a
message before anything is launched, so these run without a GPU."""
import pytest

from ramforge_b200 import (RfError, _lib, dequantize_i8, i8_matmul, norm_i8, quantize_i8, swiglu_i8, verify_drafts,
                           verify_greedy)

P = 1 << 20  # a pointer that is never followed


def refused(fn, a, kw, text):
    with pytest.raises(RfError) as e:
        fn(**{**a, **kw})
    assert e.value.code == _lib.RF_EINVAL and text in str(e.value), str(e.value)


NORM = dict(x_ptr=P, weight_ptr=P, eps=1e-5, q_ptr=P, scale_ptr=P, act_type=_lib.ACT_F32, n_rows=3, n_cols=64,
            add_ptr=P, sum_ptr=P)
SWIGLU = dict(gate_ptr=P, up_ptr=P, q_ptr=P, scale_ptr=P, act_type=_lib.ACT_F16, n_rows=3, n_cols=64)
QUANT = dict(x_ptr=P, q_ptr=P, scale_ptr=P, act_type=_lib.ACT_BF16, n_rows=3, n_cols=64)
DEQUANT = dict(q_ptr=P, scale_ptr=P, out_ptr=P, act_type=_lib.ACT_BF16, n_rows=3, n_cols=64)
ROWS = [(norm_i8, NORM), (swiglu_i8, SWIGLU), (quantize_i8, QUANT), (dequantize_i8, DEQUANT)]


@pytest.mark.parametrize("fn,a", ROWS)
@pytest.mark.parametrize("kw,text", [
    (dict(act_type=8), "activation type"), (dict(n_cols=0), "columns"), (dict(n_cols=65537), "columns"),
    (dict(n_rows=1 << 31), "too many"), (dict(q_ptr=0), "null"), (dict(scale_ptr=0), "null"),
    (dict(q_stride=63), "stride"), (dict(scale_ptr=P + 2), "scales must be 4-byte")])
def test_rows_calls_refuse(fn, a, kw, text):
    refused(fn, a, kw, text)


@pytest.mark.parametrize("fn,a,kw,text", [
    (norm_i8, NORM, dict(x_ptr=0), "null rows"), (norm_i8, NORM, dict(x_stride=60), "stride"),
    (norm_i8, NORM, dict(add_stride=1), "stride"), (norm_i8, NORM, dict(sum_stride=63), "stride"),
    (norm_i8, NORM, dict(x_ptr=P + 2), "element size"), (norm_i8, NORM, dict(add_ptr=P + 1), "element size"),
    (norm_i8, NORM, dict(sum_ptr=P + 2), "element size"), (norm_i8, NORM, dict(weight_ptr=P + 2), "norm weights"),
    (norm_i8, NORM, dict(eps=-1e-9), "eps"), (norm_i8, NORM, dict(eps=float("nan")), "eps"),
    (norm_i8, NORM, dict(eps=float("inf")), "eps"),
    (swiglu_i8, SWIGLU, dict(gate_ptr=0), "null gate"), (swiglu_i8, SWIGLU, dict(up_ptr=0), "null gate"),
    (swiglu_i8, SWIGLU, dict(gate_stride=8), "stride"), (swiglu_i8, SWIGLU, dict(up_stride=63), "stride"),
    (swiglu_i8, SWIGLU, dict(up_ptr=P + 1), "element size"),
    (quantize_i8, QUANT, dict(x_ptr=0), "null rows"), (quantize_i8, QUANT, dict(x_ptr=P + 1), "element size"),
    (quantize_i8, QUANT, dict(x_stride=1), "stride"),
    (dequantize_i8, DEQUANT, dict(out_ptr=0), "null values"), (dequantize_i8, DEQUANT, dict(out_stride=1), "stride"),
    (dequantize_i8, DEQUANT, dict(out_ptr=P + 1), "element size")])
def test_each_rows_call_refuses(fn, a, kw, text):
    refused(fn, a, kw, text)


MM = dict(x_ptr=P, x_scale_ptr=P, w_ptr=P, w_scale_ptr=P, y_ptr=P, act_type=_lib.ACT_F32, n_tokens=3, n_out=5, n_in=64)


@pytest.mark.parametrize("kw,text", [
    (dict(act_type=2), "activation type"), (dict(n_in=0), "n_in"), (dict(n_in=65537), "n_in"),
    (dict(n_tokens=(1 << 32) - 1), "too many"), (dict(n_out=(1 << 31) - 1), "too many"), (dict(x_ptr=0), "null"),
    (dict(x_scale_ptr=0), "null"), (dict(w_ptr=0), "null"), (dict(w_scale_ptr=0), "null"), (dict(y_ptr=0), "null"),
    (dict(x_stride=48), "x stride"), (dict(w_stride=48), "w stride"), (dict(x_stride=72), "x rows must be 16-byte"),
    (dict(w_stride=65), "w rows must be 16-byte"), (dict(n_in=50), "x rows must be 16-byte"),
    (dict(x_ptr=P + 8), "x rows must be 16-byte"), (dict(w_ptr=P + 4), "w rows must be 16-byte"),
    (dict(y_stride=4), "y stride"), (dict(y_ptr=P + 2), "element size"), (dict(x_scale_ptr=P + 2), "scales and bias"),
    (dict(w_scale_ptr=P + 1), "scales and bias"), (dict(bias_ptr=P + 2), "scales and bias")])
def test_matmul_refuses(kw, text):
    refused(i8_matmul, MM, kw, text)


VD = dict(target_ptr=P, draft_ptr=P, prob_type=_lib.ACT_F32, vocab=100, n_seqs=2, n_tokens=3, tokens_ptr=P,
          accept_u_ptr=P, next_u_ptr=P, out_tokens_ptr=P, n_accepted_ptr=P)
VG = dict(logits_ptr=P, logit_type=_lib.ACT_F32, vocab=100, n_seqs=2, n_tokens=3, tokens_ptr=P, best_ptr=P,
          out_tokens_ptr=P, n_accepted_ptr=P)


@pytest.mark.parametrize("fn,a", [(verify_drafts, VD), (verify_greedy, VG)])
@pytest.mark.parametrize("kw,text", [
    (dict(vocab=0), "vocabulary"), (dict(vocab=1 << 31), "vocabulary"), (dict(n_tokens=1025), "0..1024"),
    (dict(n_seqs=(1 << 32) - 1), "too many"), (dict(out_tokens_ptr=0), "null"), (dict(n_accepted_ptr=0), "null"),
    (dict(tokens_ptr=0), "null drafted"), (dict(positions_ptr=P), "hist_len"), (dict(parent_ptr=P + 2), "4-byte"),
    (dict(tokens_ptr=P + 1), "4-byte"), (dict(n_draft_ptr=P + 2), "4-byte"), (dict(hist_len_ptr=P + 3), "4-byte"),
    (dict(n_accepted_ptr=P + 2), "4-byte"), (dict(out_tokens_ptr=P + 2), "4-byte")])
def test_verdicts_refuse(fn, a, kw, text):
    refused(fn, a, kw, text)


@pytest.mark.parametrize("fn,a,kw,text", [
    (verify_drafts, VD, dict(prob_type=8), "activation type"), (verify_drafts, VD, dict(target_ptr=0), "null"),
    (verify_drafts, VD, dict(accept_u_ptr=0), "random"), (verify_drafts, VD, dict(next_u_ptr=0), "random"),
    (verify_drafts, VD, dict(target_stride=99), "stride"), (verify_drafts, VD, dict(draft_stride=99), "stride"),
    (verify_drafts, VD, dict(target_ptr=P + 2), "element size"), (verify_drafts, VD, dict(draft_ptr=P + 2), "element size"),
    (verify_drafts, VD, dict(next_u_ptr=P + 2), "random"), (verify_drafts, VD, dict(accept_u_ptr=P + 1), "random"),
    (verify_greedy, VG, dict(logit_type=8), "activation type"), (verify_greedy, VG, dict(logits_ptr=0), "null"),
    (verify_greedy, VG, dict(best_ptr=0), "null"), (verify_greedy, VG, dict(best_ptr=P + 2), "4-byte"),
    (verify_greedy, VG, dict(logits_stride=99), "stride")])
def test_each_verdict_refuses(fn, a, kw, text):
    refused(fn, a, kw, text)


def test_nothing_to_do_is_no_error():
    for fn, a in ROWS:
        fn(**{**a, "n_rows": 0})
    i8_matmul(**{**MM, "n_tokens": 0})
    i8_matmul(**{**MM, "n_out": 0})
    verify_drafts(**{**VD, "n_seqs": 0})
    verify_greedy(**{**VG, "n_seqs": 0})
