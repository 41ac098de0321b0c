"""Host side of the attention over paged caches and of the verification of drafts: refusals, before any launch (no GPU)."""
import ctypes

import pytest
import torch

from arcticinference_amd import _native, py_custom_ops as ops
from attention_helpers import make_attention_case


@pytest.fixture(scope="module")
def loaded():
    assert ops.try_load_torch_library(), "libarctic_mi355x.so is not built"
    return ops


def attention_args(**other):
    c = make_attention_case(lengths=[30, 100], new=[1, 1], heads=8, kv_heads=2, size=64)
    args = dict(query=c["query"], key_cache=c["key"], value_cache=c["value"], block_table=c["table"], seq_lens=c["seq_lens"],
                kv_cache_dtype="auto", k_scale=c["k_scale"], v_scale=c["v_scale"], scale=0.125, max_seq_len=100, window=0, num_sinks=0,
                out=torch.empty_like(c["query"]))
    args.update(other)
    return args


BAD_ATTENTION = [
    (dict(query=torch.zeros(2, 8, 64, dtype=torch.float64)), "queries must be fp32, fp16 or bf16"),
    (dict(kv_cache_dtype="nvfp4"), "Unsupported data type of kv cache: nvfp4"),
    (dict(query=torch.zeros(2, 64, dtype=torch.bfloat16)), "queries must be"),
    (dict(key_cache=torch.zeros(4, 16, 2, 32, dtype=torch.bfloat16)), "both of one shape"),
    (dict(query=torch.zeros(2, 8, 32, dtype=torch.bfloat16)), "differ in their head_size"),
    (dict(query=torch.zeros(2, 7, 64, dtype=torch.bfloat16)), "must be a multiple of the caches'"),
    (dict(query=torch.zeros(2, 8, 64, dtype=torch.float16)), "must be of the queries' type"),
    (dict(kv_cache_dtype="fp8"), "elements of one byte"),
    (dict(query=torch.zeros(2, 64, 8, dtype=torch.bfloat16).transpose(1, 2)), "last dimension of the queries"),
    (dict(out=torch.zeros(2, 8, 65, dtype=torch.bfloat16)), "out must have the queries' type and shape"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), "seq_lens must be a contiguous int32"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), "must be a contiguous int32|block_table must be int32"),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int32)), "block_table must be int32"),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int64)), "block_table must be int32"),
    (dict(block_table=torch.zeros(4, 2, dtype=torch.int32).t()), "block_table must be int32"),
    (dict(max_seq_len=-1), "max_seq_len must not be negative"),
    (dict(window=-1), "window must be positive"),
    (dict(num_sinks=-1), "num_sinks not negative"),
    (dict(), "must be CUDA tensors"),
]


@pytest.mark.parametrize("other,match", BAD_ATTENTION)
def test_attention_refuses_before_any_launch(loaded, other, match):
    args = attention_args(**other)
    with pytest.raises(RuntimeError, match=match):
        ops._IMPLS["paged_attention"](*args.values())
    if "query" in other and other["query"].dim() == 2:
        return
    start = torch.tensor([0, 1, 2], dtype=torch.int32)
    with pytest.raises(RuntimeError, match=match):
        ops._IMPLS["paged_attention_ragged"](args.pop("query"), start, *args.values())


def test_more_refusals(loaded):
    args = attention_args()
    query = args.pop("query")
    ragged = ops._IMPLS["paged_attention_ragged"]
    for bad in (torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int64), torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(RuntimeError, match="query_start must be a contiguous int32"):
            ragged(query, bad, *args.values())
    with pytest.raises(RuntimeError, match=r"queries must be \[tokens, heads, head_size\]"):
        ragged(query[None], torch.zeros(3, dtype=torch.int32), *args.values())
    fp8 = attention_args(kv_cache_dtype="fp8", key_cache=torch.zeros(4, 16, 2, 64, dtype=torch.uint8),
                         value_cache=torch.zeros(4, 16, 2, 64, dtype=torch.uint8))
    for bad in (torch.ones(1, dtype=torch.float64), torch.ones(2)):
        with pytest.raises(RuntimeError, match="float32 tensors of one element"):
            ops._IMPLS["paged_attention"](*dict(fp8, k_scale=bad).values())
    for window in (0, -3):
        with pytest.raises(ValueError, match="window must be at least 1"):
            ops.paged_attention(*list(attention_args().values())[:10], window=window)
    # no CPU path
    with pytest.raises(NotImplementedError, match="CPU"):
        ops.paged_attention(*list(attention_args().values())[:10])
    logits = torch.zeros(3, 50)
    rest = (torch.tensor([0, 3], dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int64), torch.zeros(1, 2), torch.zeros(1))
    with pytest.raises(NotImplementedError, match="CPU"):
        ops.verify_draft_tokens(logits, *rest)
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        ops._IMPLS["verify_draft_tokens"](logits, *rest, None)


def test_meta_tensors(loaded):
    args = {k: v.to("meta") if isinstance(v, torch.Tensor) else v for k, v in attention_args().items()}
    out = ops.paged_attention(*list(args.values())[:10])
    assert out.is_meta and out.shape == (2, 8, 64) and out.dtype == torch.bfloat16
    meta = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="meta")
    tokens, counts = ops.verify_draft_tokens(meta(5, 90), meta(3, dtype=torch.int32), meta(2, 4, dtype=torch.int64), meta(2, 4), meta(2))
    assert tokens.shape == (2, 5) and counts.shape == (2,) and tokens.dtype == counts.dtype == torch.int64


FAKE = ctypes.c_void_p(0x7F0000000000)   # never dereferenced: every call below is refused on its arguments


def cache(**other):
    values = dict(key_cache=FAKE.value, value_cache=FAKE.value, k_scale=FAKE.value, v_scale=FAKE.value, num_blocks=8, key_block_stride=2048,
                  key_token_stride=128, key_head_stride=64, value_block_stride=2048, value_token_stride=128, value_head_stride=64,
                  block_size=16, num_kv_heads=2, head_size=64, kv_cache_dtype=0)
    values.update(other)
    return _native.PagedCache(**values)


def abi_attention(lib, c, **other):
    a = dict(out=FAKE, query=FAKE, table=FAKE, lens=FAKE, batch=2, new=1, heads=8, max_blocks=4, table_stride=4, qt=512, qh=64, ot=512,
             oh=64, scale=1.0, most=64, window=0, sinks=0, dtype=2, ws=None, ws_bytes=0)
    a.update(other)
    return lib.arctic_paged_attention(a["out"], a["query"], ctypes.byref(c) if c else None, a["table"], a["lens"], a["batch"], a["new"],
                                      a["heads"], a["max_blocks"], a["table_stride"], a["qt"], a["qh"], a["ot"], a["oh"], a["scale"],
                                      a["most"], a["window"], a["sinks"], a["dtype"], a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("cache_other,other,code,text", [
    ({}, dict(dtype=9), 2, b"fp32, fp16 or bf16"),
    ({"kv_cache_dtype": 5}, {}, 2, b"Unsupported data type of kv cache"),
    ({"head_size": 0}, {}, 1, b"must be positive"),
    ({"block_size": -1}, {}, 1, b"must be positive"),
    ({"num_kv_heads": 3}, {}, 1, b"must be a multiple"),
    ({"head_size": 513}, {}, 2, b"at most 512"),
    ({"block_size": 1 << 21}, {}, 1, b"beyond 2^20"),
    ({"num_blocks": 1 << 40}, {}, 1, b"beyond 2^31"),
    ({}, dict(batch=-1), 1, b"negative"),
    ({}, dict(batch=1 << 20, new=1 << 20), 1, b"2^31"),
    ({}, dict(window=-1), 1, b"must not be negative"),
    ({}, dict(sinks=-1), 1, b"must not be negative"),
    ({"key_token_stride": -1}, {}, 1, b"pitch out of range"),
    ({"value_block_stride": 1 << 60}, {}, 1, b"pitch out of range"),
    ({}, dict(qt=1 << 62), 1, b"pitch out of range"),
    ({}, dict(out=None), 1, b"null tensor pointer"),
    ({}, dict(table=None), 1, b"null tensor pointer"),
    ({"key_cache": None}, {}, 1, b"null tensor pointer"),
    ({"kv_cache_dtype": 1, "k_scale": None}, {}, 1, b"needs k_scale"),
    ({}, dict(query=ctypes.c_void_p(0x7F0000000001)), 2, b"multiple of its element size"),
])
def test_abi_refuses_without_launching(loaded, cache_other, other, code, text):
    lib = _native.load()
    assert abi_attention(lib, cache(**cache_other), **other) == code
    assert text in lib.arctic_last_error(), lib.arctic_last_error()


def test_abi_empty_calls_and_missing_descriptions(loaded):
    lib = _native.load()
    assert abi_attention(lib, None) == 1 and b"null cache" in lib.arctic_last_error()
    assert abi_attention(lib, cache(), batch=0) == 0
    assert abi_attention(lib, cache(), new=0) == 0
    ragged = lambda start, total: lib.arctic_paged_attention_ragged(
        FAKE, FAKE, start, ctypes.byref(cache()), FAKE, FAKE, 2, total, 8, 4, 4, 512, 64, 512, 64, 1.0, 64, 0, 0, 2, None, 0, None)
    assert ragged(None, 5) == 1 and b"query_start is missing" in lib.arctic_last_error()
    assert ragged(None, 0) == 0


def abi_verify(lib, **other):
    a = dict(tokens=FAKE, counts=FAKE, logits=FAKE, start=FAKE, drafts=FAKE, accept=FAKE, sample=FAKE, temps=None, batch=2, most=3, rows=8,
             vocab=1000, stride=1000, ds=3, us=3, dtype=2, ws=FAKE, ws_bytes=1 << 30)
    a.update(other)
    return lib.arctic_verify_drafts(*a.values(), None)


@pytest.mark.parametrize("other,code,text", [
    (dict(dtype=7), 2, b"fp32, fp16 or bf16"), (dict(batch=-1), 1, b"batch and num_rows"), (dict(most=-1), 1, b"max_drafts"),
    (dict(most=1025), 1, b"max_drafts"), (dict(vocab=0), 1, b"vocab_size"), (dict(rows=1 << 31), 1, b"num_rows"),
    (dict(stride=-1), 1, b"pitch"), (dict(ds=1 << 60), 1, b"pitch"), (dict(tokens=None), 1, b"null"), (dict(drafts=None), 1, b"null"),
    (dict(logits=None), 1, b"null"), (dict(logits=ctypes.c_void_p(0x7F0000000001)), 2, b"element size"), (dict(ws=None), 1, b"workspace"),
    (dict(ws_bytes=8), 1, b"workspace"), (dict(batch=1 << 28, vocab=1 << 30, ws_bytes=1 << 62), 1, b"too many requests"),
])
def test_abi_verify_refuses_without_launching(loaded, other, code, text):
    lib = _native.load()
    assert abi_verify(lib, **other) == code
    assert text in lib.arctic_last_error(), lib.arctic_last_error()


def test_abi_verify_of_no_request(loaded):
    lib = _native.load()
    assert abi_verify(lib, batch=0) == 0
    assert lib.arctic_verify_drafts_workspace_bytes(0, 3, 1000, 2) == 0
    assert lib.arctic_verify_drafts_workspace_bytes(2, 3, 128256, 2) > 0


def test_an_expanded_output_is_refused(loaded):
    args = attention_args()
    args["out"] = torch.zeros(1, *args["query"].shape[1:], dtype=args["query"].dtype).expand(args["query"].shape)
    with pytest.raises(RuntimeError, match="out must not be expanded"):
        ops._IMPLS["paged_attention"](*args.values())


def test_abi_verify_of_more_requests_than_a_launch_has_lanes_for(loaded):
    lib = _native.load()
    assert abi_verify(lib, batch=1 << 24, most=0, vocab=100, ws_bytes=1 << 62) == 1
    assert b"too many requests" in lib.arctic_last_error()
