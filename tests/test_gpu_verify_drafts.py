"""Verification of drafted tokens: the tokens of the definition in 64 bits, exactly."""
import math

import pytest
import torch

from attention_helpers import verify_in_64_bits

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make_case(drafted, vocab, *, most=None, dtype=torch.bfloat16, seed=0, greedy=0.0, likely=True, pad=0, std=2.0):
    g = torch.Generator().manual_seed(seed)
    batch, most = len(drafted), max(drafted + [0]) if most is None else most
    start = [0]
    for n in drafted:
        start.append(start[-1] + n + 1)
    logits = (torch.randn(start[-1], vocab + pad, generator=g) * std).to(dtype)[:, :vocab]
    drafts = torch.randint(0, vocab, (batch, most), generator=g)
    if likely:
        for b, n in enumerate(drafted):
            for k in range(n):
                logits[start[b] + k, drafts[b, k]] = math.log(vocab) + std * std / 2 + 1.5 * torch.randn((), generator=g).item()
    temperatures = 0.6 + 0.8 * torch.rand(batch, generator=g)
    temperatures[torch.rand(batch, generator=g) < greedy] = 0.0
    return [logits, torch.tensor(start, dtype=torch.int32), drafts, torch.rand(batch, most, generator=g), torch.rand(batch, generator=g),
            temperatures]


def on_gpu(case):
    logits = case[0]
    full = torch.empty(logits.size(0), logits.stride(0), dtype=logits.dtype, device=DEV)
    full[:, :logits.size(1)].copy_(logits)
    return [full[:, :logits.size(1)]] + [None if t is None else t.to(DEV) for t in case[1:]]


def check(ops, case, what=""):
    want_tokens, want_counts = verify_in_64_bits(*case)
    tokens, counts = ops.verify_draft_tokens(*on_gpu(case))
    assert tokens.dtype == counts.dtype == torch.int64
    assert torch.equal(counts.cpu(), want_counts), f"{what}: counts {counts.tolist()} want {want_counts.tolist()}"
    assert torch.equal(tokens.cpu(), want_tokens), f"{what}: tokens {tokens.tolist()} want {want_tokens.tolist()}"
    return want_tokens, want_counts


@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 64, 255, 256, 1000, 4095, 4096, 4097, 8193, 32000, 50257, 128256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_vocabularies(ops, vocab, dtype):
    check(ops, make_case([3, 0, 2], vocab, dtype=dtype, seed=vocab))


@pytest.mark.parametrize("drafted", [[0], [1], [8], [0, 0, 0], [5, 0, 3, 1], [3] * 40, [40, 2]])
@pytest.mark.parametrize("greedy", [0.0, 0.5, 1.0])
def test_numbers_of_drafts(ops, drafted, greedy):
    _, counts = check(ops, make_case(drafted, 5000, seed=len(drafted), greedy=greedy))
    assert (counts >= 1).all()


def test_the_samples_of_many_requests(ops):
    """Hundreds of draws from rows whose borders are as narrow as they get: the 64-bit sums decide."""
    for seed in range(3):
        case = make_case([1] * 150, 30000, dtype=torch.float32, seed=seed, std=0.3, likely=False)
        _, counts = check(ops, case)
        case = make_case([2] * 100, 20000, seed=10 + seed)
        _, counts = check(ops, case)
        assert 1 <= int(counts.min()) and int(counts.max()) == 3


def test_more_places_than_drafts_and_requests_without_rows(ops):
    case = make_case([2, 4, 0], 700, most=9, seed=3)
    check(ops, case)
    case[1] = torch.tensor([0, 3, 3, 8], dtype=torch.int32)      # the second request has no row
    want, counts = check(ops, case)
    assert counts[1] == 0 and (want[1] == -1).all()
    case[1] = torch.tensor([0, 3, 200, 300], dtype=torch.int32)  # rows that are not there
    check(ops, case)
    case[1] = torch.tensor([-4, 2, 1, 2 ** 31 - 1], dtype=torch.int32)
    check(ops, case)


def test_strides(ops):
    for pad in (1, 3, 8):
        case = make_case([3, 1, 2], 3001, seed=4, pad=pad)
        wide = torch.zeros(3, 7, dtype=torch.int64)
        wide[:, :3] = case[2]
        case[2] = wide[:, :3]
        uniforms = torch.zeros(3, 5)
        uniforms[:, :3] = case[3]
        want = verify_in_64_bits(*case)
        dev = on_gpu(case)
        dev[2], dev[3] = wide.to(DEV)[:, :3], uniforms.to(DEV)[:, :3]
        got = ops.verify_draft_tokens(*dev)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_without_temperatures(ops):
    case = make_case([3, 1, 2], 3001, seed=5)
    case[5] = None
    check(ops, case)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_a_filter_has_cut(ops, dtype):
    for keep in (1, 2, 50):
        case = make_case([2] * 20, 9000, dtype=dtype, seed=6 + keep)
        top = case[0].float().topk(keep, dim=-1)
        case[0] = torch.full_like(case[0], -math.inf).scatter(1, top.indices, top.values.to(dtype))
        check(ops, case, f"{keep} kept")


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_rows_without_a_distribution(ops, bad):
    case = make_case([2, 2, 2, 0, 1], 9000, seed=7)
    case[3].zero_()                              # whatever has any weight is accepted
    case[0][0, 8500] = bad                       # request 0: its first row
    case[0][4, [100, 4500]] = bad                # request 1: its second row, twice
    case[0][5, int(case[2][1, 1])] = 1.0
    case[0][8] = -math.inf                       # request 2: the row behind its drafts
    case[0][9] = -math.inf                       # request 3: the only row
    case[0][10, int(case[2][4, 0])] = bad        # request 4: the draft itself
    want, counts = check(ops, case)
    assert counts.tolist() == [1, 2, 3, 1, 1] and want[0, 0] == 8500 and want[1, 1] == 100 and want[2, 2] == 0 and want[3, 0] == 0
    case[5].zero_()
    check(ops, case, "greedy")


def test_drafts_outside_the_vocabulary_are_not_accepted(ops):
    case = make_case([2, 2, 2], 900, seed=8)
    case[3].zero_()
    case[2][0, 0], case[2][1, 1], case[2][2, 0] = -1, 900, 2 ** 40
    _, counts = check(ops, case)
    assert counts.tolist() == [1, 2, 1]


def test_the_same_draft_twice_and_a_draft_that_holds_all_the_weight(ops):
    case = make_case([3, 3], 900, seed=9)
    case[2][0] = 5
    case[0][0:3, 5] = 20.0
    case[0][4, :] = -math.inf
    case[0][4, int(case[2][1, 0])] = 0.0
    case[3][1, 0] = 1.0                          # outside [0, 1): not accepted, and nothing else has weight
    want, _ = check(ops, case)
    assert want[1, 0] == case[2][1, 0]


def test_uniform_numbers_at_their_ends(ops):
    below = 1.0 - 2.0 ** -24
    for u, s in ((0.0, 0.0), (below, below), (0.0, below), (below, 0.0)):
        case = make_case([2, 1, 3], 5000, seed=10)
        case[3].fill_(u)
        case[4].fill_(s)
        check(ops, case, f"{u} {s}")


def test_temperatures_from_tiny_to_huge(ops):
    for t in (-1.0, 1e-30, 1e-3, 50.0, 1e30, math.inf, math.nan):
        case = make_case([2, 1, 3], 5000, seed=11)
        case[5].fill_(t)
        check(ops, case, f"temperature {t}")


def test_greedy_takes_the_lowest_index_of_equal_values(ops):
    case = make_case([2, 2], 9000, seed=12, likely=False)
    case[0].clamp_(max=1.0)
    case[5].zero_()
    first = case[0].float().argmax(-1)
    case[2][0, 0], case[2][0, 1] = first[0], first[1]
    case[2][1, 0] = (case[0][3] == 1.0).nonzero()[1]   # equal to the largest, but not the first
    _, counts = check(ops, case)
    assert counts.tolist() == [3, 1]


def test_no_request(ops):
    case = make_case([1], 100, seed=13)
    empty = [case[0], case[1][:1], case[2][:0], case[3][:0], case[4][:0], case[5][:0]]
    tokens, counts = ops.verify_draft_tokens(*on_gpu(empty))
    assert tokens.shape == (0, 2) and counts.shape == (0,)


def test_captured_and_replayed_with_other_inputs(ops):
    case = make_case([3, 1, 2, 0], 20000, seed=14, greedy=0.3)
    dev = on_gpu(case)
    ops.verify_draft_tokens(*dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, counts = ops.verify_draft_tokens(*dev)
    for seed in (15, 16, 14, 17):
        other = make_case([3, 1, 2, 0] if seed != 16 else [0, 3, 3, 0], 20000, seed=seed, most=3, greedy=0.3)
        for t, n in zip(dev, other):
            t.copy_(n)
        tokens.zero_()
        (torch.ones(1000, device=DEV) * 2).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        want = verify_in_64_bits(*other)
        assert torch.equal(tokens.cpu(), want[0]) and torch.equal(counts.cpu(), want[1])


def test_two_calls_at_once_on_two_streams(ops):
    cases = [on_gpu(make_case([3] * 20, 50257, seed=s)) for s in (18, 19)]
    want = [[t.clone() for t in ops.verify_draft_tokens(*c)] for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.verify_draft_tokens(*c))
    torch.cuda.synchronize()
    for w, results in zip(want, got):
        assert all(torch.equal(w[0], g[0]) and torch.equal(w[1], g[1]) for g in results)


def test_the_distribution_is_the_targets(ops):
    """Over a grid of both uniform numbers the first token's frequencies are the target's probabilities, whatever is
    drafted: each token's share of the n * n points is its probability but for the grid's steps (one column of n for its
    border in the first number, and one row of n for each border in the second)."""
    n, vocab = 64, 5
    logits = torch.tensor([[0.3, -1.0, 1.2, 0.0, -0.4]])
    p = torch.softmax(logits.double()[0], 0)
    grid = (torch.arange(n).float() + 0.5) / n
    rows = torch.arange(n * n + 1, dtype=torch.int32) * 2
    for draft in (2, 1):
        tokens, counts = ops.verify_draft_tokens(
            logits.expand(2 * n * n, vocab).contiguous().to(DEV), rows.to(DEV), torch.full((n * n, 1), draft, device=DEV),
            grid.repeat_interleave(n)[:, None].contiguous().to(DEV), grid.repeat(n).to(DEV), None)
        share = torch.bincount(tokens[:, 0].cpu(), minlength=vocab).double() / (n * n)
        assert ((share - p).abs() <= 2.0 / n).all(), (share, p)


def test_with_the_frameworks_own_drafts(ops):
    """argmax drafts of a speculator's logits, the bulk write, attention of the drafted tokens, verification."""
    from attention_helpers import assert_attention, attention_in_64_bits
    g = torch.Generator().manual_seed(20)
    batch, new, kv_heads, heads, size, block, vocab = 6, 4, 2, 8, 128, 16, 3000
    lengths = [200, 17, 64, 5, 130, 33]
    pages = [(n + block - 1) // block for n in lengths]
    caches = torch.zeros(2, sum(pages), block, kv_heads, size, dtype=torch.uint8, device=DEV)
    table = torch.zeros(batch, max(pages), dtype=torch.int32)
    order, at, slots = torch.randperm(sum(pages), generator=g), 0, []
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n].to(torch.int32)
        slots += [int(table[b, j // block]) * block + j % block for j in range(lengths[b])]
        at += n
    tokens = sum(lengths)
    rn = lambda *shape: torch.randn(*shape, generator=g).to(torch.bfloat16).to(DEV)
    keys, values = rn(tokens, kv_heads * size), rn(tokens, kv_heads * size)
    scale = torch.tensor([0.02], device=DEV)
    query, out_rows, head = rn(batch * new, heads, size), rn(heads * size, vocab), None
    target = rn(batch * new, vocab)

    def step():
        ops.reshape_and_cache_flash_bulk(keys, values, [caches[0]], [caches[1]], torch.tensor(slots, device=DEV), "fp8", [scale[0]],
                                         [scale[0]], kv_heads, size)
        return rest()

    table, seq_lens = table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
    row_start = torch.arange(batch + 1, dtype=torch.int32, device=DEV) * new
    uniforms = torch.rand(batch, new - 1, generator=g).to(DEV), torch.rand(batch, generator=g).to(DEV)

    def rest():
        out = ops.paged_attention(query.view(batch, new, heads, size), caches[0], caches[1], table, seq_lens, "fp8", scale, scale,
                                  1 / math.sqrt(size), max(lengths))
        logits = torch.mm(out.view(batch * new, -1), out_rows)
        drafts = ops.speculator_argmax(target, vocab).view(batch, new)[:, :new - 1].contiguous()
        return out, logits, drafts, *ops.verify_draft_tokens(logits, row_start, drafts, *uniforms)

    out, logits, drafts, got, counts = step()
    case = dict(query=query, table=table, seq_lens=seq_lens, key=caches[0], value=caches[1], kv="fp8", k_scale=scale, v_scale=scale,
                scale=1 / math.sqrt(size), new=[new] * batch, block=block)
    want, bound = attention_in_64_bits(case)
    assert_attention(out.view(batch * new, heads, size), want, bound)
    want = verify_in_64_bits(logits, row_start, drafts, *uniforms)
    assert torch.equal(got.cpu(), want[0]) and torch.equal(counts.cpu(), want[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = rest()
    for _ in range(3):
        for t in again:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(again, (out, logits, drafts, got, counts)):
            assert torch.equal(a, b)


def test_errors(ops):
    case = on_gpu(make_case([2, 1], 100, seed=21))
    for at, bad, match in ((0, case[0].double(), "fp32, fp16 or bf16"), (0, case[0][None], "vocab_size"), (0, case[0].t(), "contiguous"),
                           (1, case[1].long(), "int32"), (1, case[1][:2], "one entry more"), (2, case[2].int(), "int64"),
                           (3, case[3][:, :1], "shape"), (4, case[4].double(), "float32"), (5, case[5][:1], "one entry per request"),
                           (1, case[1].cpu(), "same device"), (5, case[5].cpu(), "same device")):
        with pytest.raises(RuntimeError, match=match):
            ops.verify_draft_tokens(*case[:at], bad, *case[at + 1:])
