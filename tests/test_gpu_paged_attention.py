"""Attention over paged caches against its definition in 64 bits."""
import math

import pytest
import torch

from attention_helpers import assert_attention, attention_in_64_bits, make_attention_case

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def cache_args(c, most=None):
    return (c["key"], c["value"], c["table"], c["seq_lens"], c["kv"], c["k_scale"], c["v_scale"], c["scale"],
            c["most"] if most is None else most)


def check(ops, c, window=None, sinks=0, out=None, most=None, ragged=True, what=""):
    """Through both entry points where every sequence has the same number of queries."""
    want, bound = attention_in_64_bits(c, window, sinks)
    visible = dict(window=window, num_sinks=sinks)
    if ragged:
        got = ops.paged_attention_ragged(c["query"], c["query_start"], *cache_args(c, most), **visible)
        assert_attention(got, want, bound, what + " ragged")
    new = set(c["new"])
    if len(new) == 1 and new != {0}:
        n = new.pop()
        query = c["query"].view(-1, n, *c["query"].shape[1:]) if c["query"].is_contiguous() else c["query"].unflatten(0, (-1, n))
        got = ops.paged_attention(query, *cache_args(c, most), **visible)
        assert got.shape == query.shape
        assert_attention(got.flatten(0, 1), want, bound, what + " uniform")
        if n == 1:
            got = ops.paged_attention(c["query"], *cache_args(c, most), **visible)
            assert_attention(got, want, bound, what + " one token")


@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (8, 2), (6, 1), (20, 4), (16, 1), (32, 1), (7, 1)])
@pytest.mark.parametrize("new", [1, 2, 5])
def test_head_groups(ops, heads, kv_heads, new):
    check(ops, make_attention_case(lengths=[61, 5, 130], new=[new] * 3, heads=heads, kv_heads=kv_heads, size=64, seed=1, device=DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kv", ["auto", "fp8", "fp8_e4m3", "fp8_e5m2"])
@pytest.mark.parametrize("size", [64, 80, 128])
def test_types(ops, dtype, kv, size):
    check(ops, make_attention_case(lengths=[200, 33], new=[3, 3], heads=8, kv_heads=2, size=size, dtype=dtype, kv=kv, seed=2, device=DEV))


@pytest.mark.parametrize("size", [1, 8, 16, 24, 40, 72, 96, 100, 112, 136, 160, 192, 200, 256, 264, 512])
@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_head_sizes(ops, size, kv):
    check(ops, make_attention_case(lengths=[70, 17], new=[2, 2], heads=4, kv_heads=2, size=size, kv=kv, seed=3, device=DEV))


@pytest.mark.parametrize("block", [1, 2, 5, 8, 16, 24, 32, 48, 64, 128, 256])
@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_block_sizes(ops, block, kv):
    """Pages that end inside a tile, tiles that span many pages."""
    c = make_attention_case(lengths=[300, 31, 257], new=[2, 2, 2], heads=8, kv_heads=2, size=128, block=block, kv=kv, seed=4, device=DEV)
    check(ops, c)
    check(ops, c, window=40, sinks=3)


@pytest.mark.parametrize("length", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000])
def test_lengths(ops, length):
    check(ops, make_attention_case(lengths=[length, 40, length], new=[1, 1, 1], heads=8, kv_heads=2, size=128, seed=5, device=DEV))


def test_sequences_shorter_than_their_queries_answer_zeros(ops):
    c = make_attention_case(lengths=[2, 0, 5, 1], new=[4, 4, 4, 4], heads=4, kv_heads=2, size=64, seed=6, device=DEV)
    check(ops, c)
    got = ops.paged_attention(c["query"].view(4, 4, 4, 64), *cache_args(c))
    assert not got[0, :2].any() and not got[1].any() and not got[3, :3].any() and bool(got[0, 2:].any())


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 5), (16, 0), (17, 4), (64, 33), (100, 1000), (1000, 2), (31, 64)])
@pytest.mark.parametrize("new", [1, 4, 90])
def test_windows_and_sinks(ops, window, sinks, new):
    check(ops, make_attention_case(lengths=[400, 95, 90], new=[new] * 3, heads=4, kv_heads=2, size=64, seed=7, device=DEV), window, sinks,
          what=f"window {window} sinks {sinks}")


@pytest.mark.parametrize("unseen", [math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).max])
@pytest.mark.parametrize("kv", ["auto", "fp8"])
@pytest.mark.parametrize("block", [16, 5])
def test_what_is_not_seen_does_not_matter(ops, unseen, kv, block):
    """Slots without a token (behind the end of a last page, in pages of no sequence) hold NaN or infinities."""
    c = make_attention_case(lengths=[37, 130, 1], new=[1, 1, 1], heads=8, kv_heads=2, size=128, kv=kv, block=block, seed=8, unseen=unseen, device=DEV)
    check(ops, c)
    check(ops, c, window=20, sinks=2)


def poison(c, positions, what):
    """Sequence 0's tokens at `positions` hold `what`, in both caches."""
    for j in positions:
        page, off = int(c["table"][0, j // c["block"]]), j % c["block"]
        for cache in (c["key"], c["value"]):
            cache[page, off] = what if c["kv"] == "auto" else 0x7F


@pytest.mark.parametrize("kv", ["auto", "fp8"])
@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("new", [3, 70])
def test_a_later_token_and_one_behind_the_window_do_not_matter(ops, kv, what, new):
    """The last token's K and V are NaN or infinite: queries before it do not see them, nor do queries whose window has
    passed a poisoned token."""
    c = make_attention_case(lengths=[170], new=[new], heads=8, kv_heads=2, size=128, kv=kv, seed=9, device=DEV)
    clean = {k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    want, bound = attention_in_64_bits(clean)
    poison(c, [169], what)
    for got in (ops.paged_attention(c["query"][None], *cache_args(c))[0],
                ops.paged_attention_ragged(c["query"], c["query_start"], *cache_args(c))):
        assert_attention(got[:-1], want[:-1], bound[:-1])
        assert not torch.isfinite(got[-1]).all()
    c = {k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in clean.items()}
    window = 20
    want, bound = attention_in_64_bits(c, window, 4)
    middle = 150 if new == 70 else 120   # for 70 queries some of them see it
    poison(c, [4, middle], what)
    for got in (ops.paged_attention(c["query"][None], *cache_args(c), window=window, num_sinks=4)[0],
                ops.paged_attention_ragged(c["query"], c["query_start"], *cache_args(c), window=window, num_sinks=4)):
        at = torch.arange(170 - new, 170, device=DEV)
        sees = (at >= middle) & (at < middle + window)
        assert_attention(got[~sees], want[~sees], bound[~sees])
        assert not torch.isfinite(got[sees]).all(-1).any()


def test_scores_of_the_types_lowest_value_and_infinite_ones(ops):
    """Keys that score -inf have no weight; keys of the type's lowest value overflow to an infinite score like any other
    product; a NaN that is seen reaches every query that sees it."""
    c = make_attention_case(lengths=[50], new=[1], heads=4, kv_heads=1, size=64, seed=10, device=DEV)
    c["query"].abs_()
    page, off = int(c["table"][0, 1]), 3
    c["key"][page, off] = -math.inf
    want, bound = attention_in_64_bits(c)
    assert torch.isfinite(want).all()
    assert_attention(ops.paged_attention(c["query"], *cache_args(c)), want, bound)
    c["key"][page, off] = torch.finfo(torch.bfloat16).min
    want, bound = attention_in_64_bits(c)
    assert_attention(ops.paged_attention(c["query"], *cache_args(c)), want, bound)
    c["key"][page, off] = math.nan
    assert torch.isnan(ops.paged_attention(c["query"], *cache_args(c))).all()


def test_pages_outside_the_cache_hold_no_keys(ops):
    c = make_attention_case(lengths=[100, 64, 40], new=[2, 2, 2], heads=8, kv_heads=2, size=128, seed=11, device=DEV)
    c["table"][0, 2] = -1
    c["table"][1, 0] = c["key"].size(0)
    c["table"][1, 3] = 2 ** 31 - 1
    c["table"][2, :] = -2 ** 31
    check(ops, c)
    check(ops, c, window=30, sinks=5)


def test_lengths_beyond_the_table_and_negative_ones(ops):
    c = make_attention_case(lengths=[100, 64, 40], new=[1, 1, 1], heads=8, kv_heads=2, size=128, seed=12, device=DEV)
    c["table"] = c["table"][:, :4].contiguous()
    c["seq_lens"].copy_(torch.tensor([2 ** 31 - 1, -5, 70]))
    c["table"][2] = c["table"][1]
    check(ops, c, most=100)


@pytest.mark.parametrize("most", [0, 1, 77, 5000, 1 << 30])
def test_the_longest_length_is_only_what_work_is_split_by(ops, most):
    c = make_attention_case(lengths=[1500, 3, 700], new=[1, 1, 1], heads=8, kv_heads=2, size=128, seed=13, device=DEV)
    check(ops, c, most=most)


@pytest.mark.parametrize("layout", ["flash", "flashinfer", "heads_first"])
@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_layouts_and_strides(ops, layout, kv):
    check(ops, make_attention_case(lengths=[90, 200], new=[2, 2], heads=8, kv_heads=2, size=64, kv=kv, layout=layout, pad=8, seed=14, device=DEV))
    # rows that are aligned to their elements only
    check(ops, make_attention_case(lengths=[90, 200], new=[2, 2], heads=8, kv_heads=2, size=64, kv=kv, layout=layout, pad=3, seed=15, device=DEV))


@pytest.mark.parametrize("offset", [1, 4, 8])
@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_caches_that_start_anywhere(ops, offset, kv):
    c = make_attention_case(lengths=[90, 200], new=[2, 2], heads=8, kv_heads=2, size=64, kv=kv, seed=16, device=DEV)
    for name in ("key", "value"):
        t = c[name]
        store = torch.zeros(t.numel() + offset, dtype=t.dtype, device=DEV)
        c[name] = store[offset:].view(t.shape)
        c[name].copy_(t)
    check(ops, c)


def test_output_of_the_callers_own_strides_and_rows_behind_the_last_sequence(ops):
    c = make_attention_case(lengths=[90, 200, 7], new=[5, 2, 0], heads=8, kv_heads=2, size=64, seed=17, device=DEV)
    want, bound = attention_in_64_bits(c)
    query = torch.cat([c["query"], torch.full((6, 8, 64), math.nan, dtype=torch.bfloat16, device=DEV)])
    store = torch.full((13, 10, 72), 3.0, dtype=torch.bfloat16, device=DEV)
    out = store[:, 1:9, 4:68]
    got = ops.paged_attention_ragged(query, c["query_start"], *cache_args(c), out=out)
    assert got is out
    assert_attention(out[:7], want, bound)
    assert (out[7:] == 3).all()
    store[:, 1:9, 4:68] = 3.0
    assert (store == 3).all()


@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_ragged_runs(ops, kv):
    """Prompts from their first token on, chunks, decode tokens, sequences without a query, in one call."""
    c = make_attention_case(lengths=[1, 33, 200, 300, 64, 129, 40], new=[1, 33, 200, 1, 0, 65, 7], heads=8, kv_heads=2, size=128, kv=kv,
                            seed=18, device=DEV)
    check(ops, c)
    check(ops, c, window=50, sinks=4)


@pytest.mark.parametrize("batch", [1, 64, 65, 300])
def test_many_sequences(ops, batch):
    lengths = [(7 * b) % 60 + 1 for b in range(batch)]
    new = [min(n, (3 * b) % 9) for b, n in enumerate(lengths)]
    check(ops, make_attention_case(lengths=lengths, new=new, heads=4, kv_heads=2, size=64, seed=19, device=DEV))


@pytest.mark.parametrize("size,dtype,kv", [(128, torch.bfloat16, "auto"), (64, torch.float16, "fp8"), (256, torch.bfloat16, "fp8_e5m2"),
                                           (80, torch.bfloat16, "auto")])
def test_prompts_of_several_tiles(ops, size, dtype, kv):
    c = make_attention_case(lengths=[520, 300], new=[520, 270], heads=3, kv_heads=1, size=size, dtype=dtype, kv=kv, seed=20, device=DEV)
    check(ops, c)
    check(ops, c, window=130, sinks=10)


@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_few_long_sequences(ops, kv):
    """The split over the length, and the join."""
    check(ops, make_attention_case(lengths=[20011, 13], new=[2, 2], heads=8, kv_heads=2, size=128, kv=kv, seed=21, device=DEV))
    check(ops, make_attention_case(lengths=[9001], new=[40], heads=4, kv_heads=1, size=64, kv=kv, seed=22, device=DEV))


@pytest.mark.parametrize("batch", [2, 5, 16, 40, 64, 65])
@pytest.mark.parametrize("longest", [600, 1500, 4000])
def test_tiles_dealt_to_workers(ops, batch, longest):
    """Sequences of equal and of very unequal lengths, so that shares fit as they are, fit when they grow, and do not."""
    g = torch.Generator().manual_seed(batch * longest)
    unequal = [longest] + torch.randint(1, longest, (batch - 1,), generator=g).tolist()
    for lengths in ([longest] * batch, unequal, [longest] + [1] * (batch - 1)):
        c = make_attention_case(lengths=lengths, new=[1] * batch, heads=4, kv_heads=2, size=64, seed=34, device=DEV)
        check(ops, c, ragged=False)


def test_a_peak_in_any_split(ops):
    """One key holds nearly all the weight: first, last, in the middle."""
    for at in (0, 2500, 4999):
        c = make_attention_case(lengths=[5000], new=[1], heads=4, kv_heads=1, size=128, seed=23, device=DEV)
        page, off = int(c["table"][0, at // 16]), at % 16
        c["key"][page, off] = (c["query"][0, 0] * 3).unsqueeze(0)
        check(ops, c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("slope", [0.004, 0.04, 0.4, -0.04])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_that_rise_and_fall_with_the_position(ops, dtype, slope, sign):
    """The running maximum moves a little or a lot with every tile, or never again."""
    c = make_attention_case(lengths=[700, 333], new=[70, 70], heads=4, kv_heads=2, size=64, dtype=dtype, seed=31, std=0.25, device=DEV)
    c["query"] += 0.5
    c["scale"] *= sign
    for b, n in enumerate(c["lengths"]):
        j = torch.arange(n, device=DEV)
        at = c["table"][b].long()[j // 16], j % 16
        c["key"][at] += (sign * slope * j).to(dtype)[:, None, None]
    check(ops, c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 4, 20])
def test_a_negative_scale_and_none(ops, dtype, new):
    for scale in (-0.2, 0.0):
        c = make_attention_case(lengths=[150, 900], new=[new] * 2, heads=4, kv_heads=2, size=64, dtype=dtype, seed=32, device=DEV)
        c["scale"] = scale
        check(ops, c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths,new", [([40, 7], 1), ([3000, 900], 3), ([3000, 900], 150)])
def test_the_output_may_be_the_queries(ops, dtype, lengths, new):
    c = make_attention_case(lengths=lengths, new=[new] * 2, heads=8, kv_heads=2, size=64, dtype=dtype, seed=33, device=DEV)
    want = ops.paged_attention_ragged(c["query"], c["query_start"], *cache_args(c))
    query = c["query"].clone()
    assert ops.paged_attention_ragged(query, c["query_start"], *cache_args(c), out=query) is query
    assert torch.equal(query, want)
    want = ops.paged_attention(c["query"].view(2, new, 8, 64), *cache_args(c))
    query = c["query"].clone().view(2, new, 8, 64)
    ops.paged_attention(query, *cache_args(c), out=query)
    assert torch.equal(query, want)


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 8), (torch.float32, 5)])
def test_more_rows_than_a_launch_has_lanes_for(ops, dtype, size):
    """2.4 million sequences of one token, 8 heads of which a wave or a workgroup answers each: more than 2^32 lanes."""
    batch, heads = 2_400_001, 8
    query = torch.ones(batch, heads, size, dtype=dtype, device=DEV)
    cache = torch.arange(64 * 16 * heads * size, device=DEV).remainder(251).to(dtype).view(64, 16, heads, size)
    table = torch.arange(batch, device=DEV, dtype=torch.int32).remainder(64)[:, None]
    lens = torch.ones(batch, dtype=torch.int32, device=DEV)
    one = torch.ones(1, device=DEV)
    got = ops.paged_attention(query, cache, cache, table, lens, "auto", one, one, 0.1, 1)
    assert torch.equal(got, cache[:, 0][table[:, 0].long()])
    start = torch.arange(batch + 1, dtype=torch.int32, device=DEV)
    got = ops.paged_attention_ragged(query, start, cache, cache, table, lens, "auto", one, one, 0.1, 1)
    assert torch.equal(got, cache[:, 0][table[:, 0].long()])


def test_no_sequence_and_no_query(ops):
    c = make_attention_case(lengths=[30], new=[1], heads=4, kv_heads=2, size=64, seed=24, device=DEV)
    empty = torch.empty(0, dtype=torch.int32, device=DEV)
    args = (c["key"], c["value"], c["table"][:0], empty, "auto", c["k_scale"], c["v_scale"], 0.125, 30)
    assert ops.paged_attention(c["query"][:0], *args).shape == (0, 4, 64)
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full_like(c["query"], 5.0)
    ops.paged_attention_ragged(c["query"], start, *args, out=out)
    assert (out == 5).all()
    assert ops.paged_attention(c["query"][:, None][:, :0], *cache_args(c)).shape == (1, 0, 4, 64)
    # a cache without a block, a table without a column
    none = c["key"][:0]
    got = ops.paged_attention(c["query"], none, none, c["table"], c["seq_lens"], "auto", c["k_scale"], c["v_scale"], 0.125, 30)
    assert not got.any()
    got = ops.paged_attention(c["query"], c["key"], c["value"], c["table"][:, :0], c["seq_lens"], "auto", c["k_scale"], c["v_scale"], 0.125, 30)
    assert not got.any()


def test_results_do_not_vary(ops):
    c = make_attention_case(lengths=[5000, 300, 77], new=[3, 3, 3], heads=8, kv_heads=2, size=128, seed=25, device=DEV)
    first = ops.paged_attention(c["query"].view(3, 3, 8, 128), *cache_args(c))
    again = [ops.paged_attention(c["query"].view(3, 3, 8, 128), *cache_args(c)) for _ in range(5)]
    assert all(torch.equal(first, a) for a in again)
    ragged = [ops.paged_attention_ragged(c["query"], c["query_start"], *cache_args(c)) for _ in range(5)]
    assert all(torch.equal(ragged[0], a) for a in ragged)


def test_two_calls_at_once_on_two_streams(ops):
    cases = [make_attention_case(lengths=[6000, 4000], new=[2, 2], heads=8, kv_heads=2, size=128, seed=s, device=DEV) for s in (26, 27)]
    want = [ops.paged_attention(c["query"].view(2, 2, 8, 128), *cache_args(c)) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attention(c["query"].view(2, 2, 8, 128), *cache_args(c)))
    torch.cuda.synchronize()
    for w, results in zip(want, got):
        assert all(torch.equal(w, g) for g in results)


def test_captured_and_replayed_with_other_lengths(ops):
    """A graph sees the lengths, tables and scales of its replay."""
    c = make_attention_case(lengths=[3000, 200], new=[1, 1], heads=8, kv_heads=2, size=128, kv="fp8", seed=28, device=DEV)
    ops.paged_attention(c["query"], *cache_args(c))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention(c["query"], *cache_args(c))
        out2 = ops.paged_attention_ragged(c["query"], c["query_start"], *cache_args(c))
    for lengths, scale in (([3000, 200], 0.021), ([17, 208], 0.021), ([2999, 1], 0.05), ([3000, 200], 0.021)):
        c["seq_lens"].copy_(torch.tensor(lengths, dtype=torch.int32))
        c["k_scale"].fill_(scale)
        c["lengths"] = lengths
        want, bound = attention_in_64_bits(c)
        out.zero_()
        out2.zero_()
        (torch.ones(1000, device=DEV) * 2).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        assert_attention(out, want, bound, f"replay of {lengths}")
        assert_attention(out2, want, bound, f"replay of {lengths}, ragged")


def test_through_the_dispatcher(ops):
    c = make_attention_case(lengths=[30, 100], new=[1, 1], heads=8, kv_heads=2, size=128, seed=29, device=DEV)
    want, bound = attention_in_64_bits(c)
    out = torch.empty_like(c["query"])
    torch.ops.arctic_inference.paged_attention(c["query"], *cache_args(c), 0, 0, out)
    assert_attention(out, want, bound)
    torch.ops.arctic_inference.paged_attention_ragged(c["query"], c["query_start"], *cache_args(c), 0, 0, out.zero_())
    assert_attention(out, want, bound)


def test_offsets_beyond_32_bits(ops):
    """A cache whose pages lie more than 2^32 bytes apart."""
    block, kv_heads, size = 16, 8, 128
    pages = (5 << 30) // (block * kv_heads * size * 2)
    cache = torch.zeros(pages, block, kv_heads, size, dtype=torch.bfloat16, device=DEV)
    c = make_attention_case(lengths=[70], new=[2], heads=8, kv_heads=8, size=128, seed=30, device=DEV)
    far = torch.tensor([pages - 1, 3, pages // 2, pages - 2, 0], dtype=torch.int32, device=DEV)
    value = torch.zeros_like(cache)
    for i, page in enumerate(far.tolist()):
        cache[page] = c["key"][int(c["table"][0, i])]
        value[page] = c["value"][int(c["table"][0, i])]
    c["key"], c["value"] = cache, value
    c["table"] = far[None].contiguous()
    check(ops, c)


def test_errors(ops):
    c = make_attention_case(lengths=[30, 100], new=[1, 1], heads=8, kv_heads=2, size=128, seed=31, device=DEV)
    good = [c["query"], *cache_args(c)]
    call = lambda **other: ops.paged_attention(*[other.get(str(i), a) for i, a in enumerate(good)],
                                               **{k: v for k, v in other.items() if not k.isdigit()})
    for match, other in (("must be CUDA|same device", {"4": c["seq_lens"].cpu()}), ("same device", {"1": c["key"].cpu()}),
                         ("same device", {"out": torch.empty_like(c["query"], device="cpu")}),
                         ("out must have the queries' type", {"out": c["query"].float()}),
                         ("contiguous", {"out": torch.empty(2, 128, 8, dtype=torch.bfloat16, device=DEV).transpose(1, 2)})):
        with pytest.raises(RuntimeError, match=match):
            call(**other)
    wide = torch.zeros(1, 16, 1, 520, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="head_size must be at most 512"):
        ops.paged_attention(wide[0, :2], wide, wide, c["table"], c["seq_lens"], "auto", c["k_scale"], c["v_scale"], 1.0, 100)


def test_random_configurations(ops):
    import random
    rnd = random.Random(40)
    for it in range(60):
        kv_heads, group = rnd.choice([1, 2, 3, 8]), rnd.choice([1, 2, 4, 5, 8, 16])
        size, block = rnd.choice([8, 64, 80, 96, 128, 128, 256]), rnd.choice([1, 8, 16, 16, 32, 48, 128])
        batch, most = rnd.choice([1, 2, 5, 9]), rnd.choice([3, 40, 300, 900])
        lengths = [rnd.randint(0, most) for _ in range(batch)]
        same = rnd.random() < 0.5
        new = [rnd.choice([1, 2, 4])] * batch if same else [rnd.randint(0, min(n, 150)) for n in lengths]
        if not same and sum(new) == 0:
            continue
        dtype, kv = rnd.choice([torch.bfloat16, torch.float16]), rnd.choice(["auto", "fp8", "fp8_e5m2"])
        window, sinks = rnd.choice([(None, 0), (rnd.randint(1, 200), rnd.choice([0, 1, 4, 40]))])
        layout = rnd.choice(["flash", "flashinfer", "heads_first"])
        what = f"configuration {it}: {lengths} {new} {kv_heads}x{group} {size} {block} {dtype} {kv} {window} {sinks} {layout}"
        c = make_attention_case(lengths=lengths, new=new, heads=kv_heads * group, kv_heads=kv_heads, size=size, block=block, dtype=dtype,
                                kv=kv, seed=600 + it, layout=layout, unseen=math.nan, device=DEV)
        check(ops, c, window, sinks, most=rnd.choice([None, 10, 4000]), what=what)
