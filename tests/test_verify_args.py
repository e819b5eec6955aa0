"""Refusals of the drafted-token verification calls: wrong arguments give RF_EINVAL or
RF_EUNSUPPORTED with a message before anything is launched, so these run without a GPU."""
import pytest

from ramforge_b200 import KvView, RfError, _lib, kv_cache_read, kv_cache_write, qk_norm_rope, tree_attention

P = 1 << 20  # a pointer that is never followed


def view(**kw):
    a = dict(type=_lib.TYPE_Q8_0, k_ptr=P, v_ptr=P, k_scale_ptr=P, v_scale_ptr=P, n_seqs=2, n_kv_heads=4, head_dim=128,
             capacity=64)
    a.update(kw)
    return KvView(**a)


def refused(fn, a, kw, code, text):
    with pytest.raises(RfError) as e:
        fn(**{**a, **kw})
    assert e.value.code == code and text in str(e.value), str(e.value)


NR = dict(q_ptr=P, k_ptr=P, q_out_ptr=P, k_out_ptr=P, act_type=_lib.ACT_F32, n_tokens=3, n_heads=8, n_kv_heads=2,
          head_dim=128, rope_ptr=P, rope_len=10, positions_ptr=P)


@pytest.mark.parametrize("kw,text", [
    (dict(act_type=2), "activation type"), (dict(q_ptr=0), "null queries"), (dict(q_out_ptr=0), "null queries"),
    (dict(n_heads=0), "null queries"), (dict(k_ptr=0), "null keys"), (dict(k_out_ptr=0), "null keys"),
    (dict(head_dim=127), "even number"), (dict(head_dim=0), "even number"), (dict(head_dim=258), "even number"),
    (dict(rot_dim=130), "rot_dim"), (dict(rot_dim=3), "rot_dim"), (dict(rope_ptr=0), "rotation table"),
    (dict(positions_ptr=0), "rotation table"), (dict(rope_len=0), "rotation table"), (dict(rope_ptr=P + 4), "8-byte"),
    (dict(q_ptr=P + 2), "element size"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(q_stride=1023), "stride"), (dict(k_out_stride=255), "stride"), (dict(n_tokens=1 << 30), "too many")])
def test_norm_rope_refuses(kw, text):
    refused(qk_norm_rope, NR, kw, _lib.RF_EINVAL, text)


KV = dict(cache=None, act_type=_lib.ACT_F16, n_rows=3, pos_ptr=P)


@pytest.mark.parametrize("fn,ptrs", [(kv_cache_write, ("k_ptr", "v_ptr")), (kv_cache_read, ("k_out_ptr", "v_out_ptr"))])
@pytest.mark.parametrize("kw,code,text", [
    (dict(cache=view(type=_lib.TYPE_Q4_K)), _lib.RF_EUNSUPPORTED, "neither F16 nor Q8_0"),
    (dict(cache=view(k_ptr=0)), _lib.RF_EINVAL, "null K/V cache"),
    (dict(cache=view(n_seqs=0)), _lib.RF_EINVAL, "empty"), (dict(cache=view(capacity=0)), _lib.RF_EINVAL, "empty"),
    (dict(cache=view(head_dim=48)), _lib.RF_EINVAL, "multiple of 32"),
    (dict(cache=view(head_dim=288)), _lib.RF_EINVAL, "multiple of 32"),
    (dict(cache=view(v_scale_ptr=0)), _lib.RF_EINVAL, "scale planes"),
    (dict(cache=view(v_ptr=P + 8)), _lib.RF_EINVAL, "aligned"),
    (dict(cache=view(k_scale_ptr=P + 2)), _lib.RF_EINVAL, "aligned"),
    (dict(act_type=8), _lib.RF_EINVAL, "activation type"), (dict(pos_ptr=0), _lib.RF_EINVAL, "null positions"),
    (dict(k_stride=500), _lib.RF_EINVAL, "stride"), (dict(v_stride=516), _lib.RF_EINVAL, "16 bytes"),
    (dict(n_rows=1 << 30), _lib.RF_EINVAL, "too many")])
def test_cache_calls_refuse(fn, ptrs, kw, code, text):
    refused(fn, {**KV, "cache": view(), **dict.fromkeys(ptrs, P)}, kw, code, text)


def test_cache_calls_refuse_null_and_unaligned_rows():
    refused(kv_cache_write, {**KV, "cache": view(), "k_ptr": P, "v_ptr": 0}, {}, _lib.RF_EINVAL, "null K/V rows")
    refused(kv_cache_read, {**KV, "cache": view(), "k_out_ptr": 0, "v_out_ptr": 0}, {}, _lib.RF_EINVAL,
            "null destinations")
    refused(kv_cache_write, {**KV, "cache": view(), "k_ptr": P + 8, "v_ptr": P}, {}, _lib.RF_EINVAL, "16-byte aligned")


TA = dict(q_ptr=P, out_ptr=P, act_type=_lib.ACT_BF16, n_seqs=2, n_tokens=5, n_heads=8, hist_len_ptr=P)


@pytest.mark.parametrize("kw,code,text", [
    (dict(cache=view(head_dim=96)), _lib.RF_EUNSUPPORTED, "head_dim 64 and 128"),
    (dict(cache=view(type=_lib.TYPE_F32)), _lib.RF_EUNSUPPORTED, "neither F16 nor Q8_0"),
    (dict(act_type=7), _lib.RF_EINVAL, "activation type"), (dict(q_ptr=0), _lib.RF_EINVAL, "null"),
    (dict(out_ptr=0), _lib.RF_EINVAL, "null"), (dict(hist_len_ptr=0), _lib.RF_EINVAL, "null"),
    (dict(n_seqs=3), _lib.RF_EINVAL, "the cache holds 2"), (dict(n_tokens=0), _lib.RF_EINVAL, "1..1024"),
    (dict(n_tokens=1025), _lib.RF_EINVAL, "1..1024"), (dict(n_heads=6), _lib.RF_EINVAL, "no multiple"),
    (dict(n_heads=0), _lib.RF_EINVAL, "no multiple"),
    (dict(n_heads=4 * 1025), _lib.RF_EUNSUPPORTED, "at most 1024"), (dict(scale=-0.1), _lib.RF_EINVAL, "scale"),
    (dict(scale=float("nan")), _lib.RF_EINVAL, "scale"), (dict(scale=float("inf")), _lib.RF_EINVAL, "scale"),
    (dict(q_stride=1000), _lib.RF_EINVAL, "stride"), (dict(out_stride=1028), _lib.RF_EINVAL, "16-byte"),
    (dict(q_ptr=P + 2), _lib.RF_EINVAL, "16-byte")])
def test_tree_attention_refuses(kw, code, text):
    refused(tree_attention, {"cache": view(), **TA}, kw, code, text)


def test_nothing_to_do_is_no_error():
    qk_norm_rope(**{**NR, "n_tokens": 0})
    kv_cache_write(cache=view(), k_ptr=0, v_ptr=0, act_type=_lib.ACT_F32, n_rows=0, pos_ptr=0)
    kv_cache_read(cache=view(), k_out_ptr=0, v_out_ptr=0, act_type=_lib.ACT_F32, n_rows=0, pos_ptr=0)
    tree_attention(cache=view(), **{**TA, "n_seqs": 0})
