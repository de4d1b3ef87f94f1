"""Host side of rope_and_cache, chunk_attention and verify_draft_tokens: inference, refusals, planning (no GPU)."""
import inspect
import os

import pytest
import torch
import yaml

import ms_custom_ops_b200 as ops
from ms_custom_ops_b200 import TensorSpec as T
from ms_custom_ops_b200 import _abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OPS = ("rope_and_cache", "chunk_attention", "verify_draft_tokens")


@pytest.mark.parametrize("op", OPS)
def test_signatures_agree(op):
    reg = ops.registered_ops()[op]
    y = yaml.safe_load(open(os.path.join(ROOT, "ms_custom_ops_b200", "ops", "c_api", op, op + "_op.yaml")))
    parts = []
    for name, spec in y[op]["args"].items():
        default = spec.get("default")
        default = {"false": False, "true": True}.get(default, default) if isinstance(default, str) else default
        parts.append(name if "default" not in spec else f"{name}={default}")
    assert reg == f"{op}({', '.join(parts)})"
    sig = inspect.signature(getattr(ops, op))
    assert reg == f"{op}(" + ", ".join(n if p.default is inspect._empty else f"{n}={p.default}"
                                       for n, p in sig.parameters.items()) + ")"


# ------------------------------------------------------------------------------------------ rope_and_cache
def rope_args(**kw):
    a = dict(query=T((6, 8, 128), "bfloat16"), key=T((6, 2, 128), "bfloat16"), value=T((6, 2, 128), "bfloat16"),
             key_cache=T((9, 16, 2, 128), "bfloat16"), value_cache=T((9, 16, 2, 128), "bfloat16"),
             slot_mapping=T((6,), "int32"), positions=T((6,), "int32"), cos_sin=T((100, 64), "float32"))
    a.update(kw)
    return a


def test_rope_infer():
    assert ops.rope_and_cache_infer(**rope_args()) == ((6, 8, 128), "bfloat16")
    hm = T((9, 2, 16, 128), "bfloat16")
    assert ops.rope_and_cache_infer(**rope_args(key_cache=hm, value_cache=hm, input_layout=1))[0] == (6, 8, 128)
    c8, ch = T((9, 16, 2, 128), "int8"), T((256,), "float32")
    assert ops.rope_and_cache_infer(**rope_args(key_cache=c8, value_cache=c8, k_descale=ch, v_descale=ch,
                                                k_offset=T((256,), "int32")))[1] == "bfloat16"
    assert ops.rope_and_cache_infer(**rope_args(query=T((6, 0, 128), "bfloat16")))[0] == (6, 0, 128)


@pytest.mark.parametrize("kw,error", [
    (dict(key_cache=None), ValueError),
    (dict(query=None), ValueError),
    (dict(query=T((5, 8, 128), "bfloat16")), ValueError),
    (dict(query=T((6, 8, 64), "bfloat16")), ValueError),
    (dict(query=T((6, 1024), "bfloat16")), ValueError),
    (dict(query=T((6, 8, 128), "float16")), TypeError),
    (dict(key=T((6, 2, 128), "float32")), TypeError),
    (dict(value=T((6, 4, 128), "bfloat16")), ValueError),
    (dict(value_cache=T((9, 16, 2, 64), "bfloat16")), ValueError),
    (dict(value_cache=T((9, 16, 2, 128), "int8")), TypeError),
    (dict(key_cache=T((9, 16, 2, 128), "float16"), value_cache=T((9, 16, 2, 128), "float16")), TypeError),
    (dict(key_cache=T((9, 16, 2, 128), "int8"), value_cache=T((9, 16, 2, 128), "int8")), ValueError),  # no scales
    (dict(k_descale=T((256,), "float32")), ValueError),  # scales without an int8 cache
    (dict(slot_mapping=T((6,), "int64")), TypeError),
    (dict(slot_mapping=T((7,), "int32")), ValueError),
    (dict(positions=T((5,), "int32")), ValueError),
    (dict(positions=None), ValueError),
    (dict(cos_sin=T((100, 63), "float32")), ValueError),
    (dict(cos_sin=T((100, 130), "float32")), ValueError),
    (dict(cos_sin=T((100, 64), "bfloat16")), TypeError),
    (dict(cos_sin=T((100,), "float32")), ValueError),
    (dict(q_weight=T((64,), "bfloat16")), ValueError),
    (dict(k_weight=T((128,), "float32")), TypeError),
    (dict(eps=-1.0), ValueError),
    (dict(eps=float("nan")), ValueError),
    (dict(input_layout=2), ValueError),
    (dict(oob_count=T((2,), "int32")), ValueError),
    (dict(key_cache=T((0, 16, 2, 128), "bfloat16"), value_cache=T((0, 16, 2, 128), "bfloat16")), ValueError),
])
def test_rope_refusals(kw, error):
    with pytest.raises(error):
        ops.rope_and_cache_infer(**rope_args(**kw))


def test_rope_strides():
    rows = torch.zeros(6, 12, 128, dtype=torch.bfloat16)
    ok = rope_args(query=rows[:, :8], key=rows[:, 8:10], value=rows[:, 10:])
    assert ops.rope_and_cache_infer(**ok)[0] == (6, 8, 128)
    for bad in (rows[:, ::2][:, :4], rows.transpose(0, 1)[:6], torch.zeros(6, 8, 256, dtype=torch.bfloat16)[..., ::2],
                rows[:1].expand(6, 12, 128)[:, :8]):
        with pytest.raises(RuntimeError):
            ops.rope_and_cache_infer(**rope_args(query=bad))


def test_rope_kernel_library_refuses():
    d = _abi.MscoRopeDesc()
    with pytest.raises(_abi.MscoError):
        _abi.check(_abi.lib().msco_rope_and_cache(None, *[None] * 17))
    d.dtype = d.cache_dtype = _abi.DTYPE_BF16
    d.num_q_heads, d.num_kv_heads, d.head_dim, d.rotary_dim, d.block_size = 4, 2, 128, 64, 16
    d.num_blocks, d.num_tokens, d.max_positions = 3, 2, 10
    d.q_stride, d.k_stride, d.v_stride = 512, 256, 256
    for field, bad in (("dtype", _abi.DTYPE_F32), ("cache_dtype", _abi.DTYPE_F16), ("num_kv_heads", 0), ("head_dim", 513),
                       ("rotary_dim", 63), ("rotary_dim", 130), ("block_size", 0), ("cache_layout", 2), ("q_stride", 511),
                       ("num_tokens", -1), ("eps", -1.0), ("max_positions", 10)):  # (the last: NULL tensors)
        keep = getattr(d, field)
        setattr(d, field, bad)
        with pytest.raises(_abi.MscoError):
            _abi.check(_abi.lib().msco_rope_and_cache(d, *[None] * 17))
        setattr(d, field, keep)
    d.num_tokens = 0
    _abi.check(_abi.lib().msco_rope_and_cache(d, *[None] * 17))


# ------------------------------------------------------------------------------------------ chunk_attention
def chunk_args(**kw):
    a = dict(query=T((40, 8, 128), "bfloat16"), key_cache=T((50, 16, 2, 128), "bfloat16"),
             value_cache=T((50, 16, 2, 128), "bfloat16"), block_tables=T((3, 8), "int32"), q_seq_lens=[1, 0, 30],
             context_lens=[100, 5, 30])
    a.update(kw)
    return a


def test_chunk_infer():
    assert ops.chunk_attention_infer(**chunk_args()) == ((40, 8, 128), "bfloat16")
    assert ops.chunk_attention_infer(**chunk_args(context_lens=[0, 0, 10])) == ((40, 8, 128), "bfloat16")
    assert ops.chunk_attention_infer(**chunk_args(q_seq_lens=torch.tensor([40, 0, 0], dtype=torch.int32)))[0] == (40, 8, 128)


@pytest.mark.parametrize("kw,error", [
    (dict(query=T((40, 1024), "bfloat16")), ValueError),
    (dict(query=T((40, 7, 128), "bfloat16")), ValueError),
    (dict(query=T((40, 8, 64), "bfloat16")), ValueError),
    (dict(query=T((40, 8, 128), "float16")), TypeError),
    (dict(query=T((40, 8, 128), "float32")), TypeError),
    (dict(key_cache=T((50, 16, 2, 128), "int8")), TypeError),
    (dict(key_cache=T((50, 16, 2, 320), "bfloat16"), value_cache=T((50, 16, 2, 320), "bfloat16"),
          query=T((40, 8, 320), "bfloat16")), ValueError),
    (dict(block_tables=T((3, 8), "int64")), TypeError),
    (dict(block_tables=T((8,), "int32")), ValueError),
    (dict(block_tables=None), ValueError),
    (dict(q_seq_lens=[1, 0]), ValueError),
    (dict(q_seq_lens=[20, 0, 21]), ValueError),       # more than query holds
    (dict(q_seq_lens=[1, -1, 3]), ValueError),
    (dict(context_lens=[100, -5, 30]), ValueError),
    (dict(context_lens=[129, 5, 30]), ValueError),    # behind the block table
    (dict(context_lens=[100, 5]), ValueError),
    (dict(context_lens=None), ValueError),
    (dict(q_seq_lens=T((3,), "int32")), RuntimeError),  # not on the host
    (dict(q_seq_lens=torch.tensor([1, 0, 3])), TypeError),  # int64
    (dict(window_size=-1), ValueError),
    (dict(input_layout=5), ValueError),
    (dict(qk_scale=float("inf")), ValueError),
    (dict(k_descale=T((256,), "float32")), ValueError),
    (dict(oob_count=T((1,), "int64")), TypeError),
])
def test_chunk_refusals(kw, error):
    with pytest.raises(error):
        ops.chunk_attention_infer(**chunk_args(**kw))


def test_chunk_workspace():
    # rows that are not split need none; a long context with few rows is split and does
    assert ops.chunk_attention_workspace_size(**chunk_args()) == 0
    long = chunk_args(block_tables=T((3, 4000), "int32"), context_lens=[60000, 5, 30])
    need = ops.chunk_attention_workspace_size(**long)
    assert need > 0
    # a sequence's splits do not depend on the others
    alone = ops.chunk_attention_workspace_size(**chunk_args(block_tables=T((1, 4000), "int32"), q_seq_lens=[1],
                                                            context_lens=[60000]))
    assert alone == need
    # the general kernel never splits
    odd = T((50, 16, 2, 80), "bfloat16")
    assert ops.chunk_attention_workspace_size(**chunk_args(query=T((40, 8, 80), "bfloat16"), key_cache=odd, value_cache=odd,
                                                           block_tables=T((3, 4000), "int32"), context_lens=[60000, 5, 30])) == 0


def test_chunk_plans_of_any_lengths():
    rng = torch.Generator().manual_seed(1)
    for _ in range(200):
        b = int(torch.randint(1, 8, (1,), generator=rng))
        q = torch.randint(0, 3000, (b,), generator=rng, dtype=torch.int32)
        ctx = torch.randint(0, 60000, (b,), generator=rng, dtype=torch.int32)
        size = ops.chunk_attention_workspace_size(
            T((int(q.sum()), 32, 128), "float16"), T((50, 128, 8, 128), "float16"), T((50, 128, 8, 128), "float16"),
            T((b, 500), "int32"), q, ctx, window_size=int(torch.randint(0, 2, (1,), generator=rng)) * 777)
        assert 0 <= size < 8 << 30


def test_calls_need_cuda_tensors():
    q, c = torch.zeros(4, 8, 128, dtype=torch.bfloat16), torch.zeros(5, 16, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.chunk_attention(q, c, c, torch.zeros(1, 2, dtype=torch.int32), [4], [4])
    with pytest.raises(RuntimeError):
        ops.rope_and_cache(q, q[:, :2], q[:, :2], c, c, torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32),
                           torch.zeros(9, 128))
    with pytest.raises(TypeError):
        ops.chunk_attention(None, c, c, torch.zeros(1, 2, dtype=torch.int32), [4], [4])


# ------------------------------------------------------------------------------------------ verify_draft_tokens
def verify_args(**kw):
    a = dict(target_probs=T((3, 5, 100), "float32"), draft_probs=T((3, 4, 100), "float32"), draft_tokens=T((3, 4), "int32"),
             uniform=T((3, 5), "float32"))
    a.update(kw)
    return a


def test_verify_infer():
    assert ops.verify_draft_tokens_infer(**verify_args()) == ((3, 5), "int32")
    assert ops.verify_draft_tokens_infer(**verify_args(draft_probs=None, draft_lens=T((3,), "int32"))) == ((3, 5), "int32")
    assert ops.verify_draft_tokens_infer(T((3, 1, 7), "float16"), None, T((3, 0), "int32"), T((3, 1), "float32"))[0] == (3, 1)


@pytest.mark.parametrize("kw,error", [
    (dict(target_probs=None), ValueError),
    (dict(target_probs=T((3, 4, 100), "float32")), ValueError),
    (dict(target_probs=T((3, 5, 0), "float32")), ValueError),
    (dict(target_probs=T((3, 5, 100), "int32")), TypeError),
    (dict(draft_probs=T((3, 4, 99), "float32")), ValueError),
    (dict(draft_probs=T((3, 4, 100), "float16")), TypeError),
    (dict(draft_tokens=T((3, 4), "int64")), TypeError),
    (dict(draft_tokens=T((12,), "int32")), ValueError),
    (dict(uniform=T((3, 4), "float32")), ValueError),
    (dict(uniform=T((3, 5), "float16")), TypeError),
    (dict(draft_lens=T((2,), "int32")), ValueError),
    (dict(draft_lens=T((3,), "float32")), TypeError),
])
def test_verify_refusals(kw, error):
    with pytest.raises(error):
        ops.verify_draft_tokens_infer(**verify_args(**kw))
