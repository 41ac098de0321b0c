"""Cases and the definition in 64 bits for the attention over paged caches and for the verification of drafts."""
from __future__ import annotations

import math

import numpy as np
import torch

FP8 = {"fp8": torch.float8_e4m3fn, "fp8_e4m3": torch.float8_e4m3fn, "fp8_e5m2": torch.float8_e5m2}


def make_attention_case(*, lengths, new, heads, kv_heads, size, block=16, dtype=torch.bfloat16, kv="auto", seed=0,
                        layout="flash", std=1.5, pad=0, spare=3, unseen=None, device="cpu"):
    """A cache with every sequence's pages in random order, queries, and the arguments of a call.  `new`: queries of each
    sequence.  layout "flash": [2, blocks, block, heads, size]; "flashinfer": [blocks, 2, ...]; "heads_first":
    [2, blocks, heads, block, size].  `unseen`: what slots that hold no token are filled with."""
    g = torch.Generator().manual_seed(seed)
    batch = len(lengths)
    pages = [(n + block - 1) // block for n in lengths]
    total = sum(pages) + spare
    shape = {"flash": (2, total, block, kv_heads, size), "flashinfer": (total, 2, block, kv_heads, size),
             "heads_first": (2, total, kv_heads, block, size)}[layout]
    values = torch.randn(shape, generator=g)
    scales = (torch.tensor([0.021]), torch.tensor([0.013]))
    if kv == "auto":
        buf = values.to(dtype)
    else:
        scale = torch.tensor([s.item() for s in scales])
        at = [1] * 5
        at[1 if layout == "flashinfer" else 0] = 2
        buf = (values / scale.view(at)).to(FP8[kv]).view(torch.uint8)
    views = {"flash": lambda: (buf[0], buf[1]), "flashinfer": lambda: (buf[:, 0], buf[:, 1]),
             "heads_first": lambda: (buf[0].transpose(1, 2), buf[1].transpose(1, 2))}[layout]
    key, value = views()
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((batch, max(pages + [1]) + 2), -7, dtype=torch.int32)
    at = 0
    used = torch.zeros(total, block, dtype=torch.bool)
    for b, n in enumerate(pages):
        mine = order[at:at + n]
        table[b, :n] = mine
        at += n
        for i, page in enumerate(mine.tolist()):
            used[page, :max(0, min(block, lengths[b] - i * block))] = True
    if unseen is not None:
        for cache in (key, value):
            cache[~used] = torch.tensor(unseen).to(cache.dtype) if kv == "auto" else torch.tensor(0x7F, dtype=torch.uint8)
    tokens = sum(new)
    query = (torch.randn(tokens, heads, size + pad, generator=g) * std).to(dtype)[..., :size]
    start = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
    move = lambda t: t.to(device)
    buf = move(buf)
    key, value = views()
    return dict(query=query if device == "cpu" else move(query), query_start=move(start), key=key, value=value, table=move(table),
                seq_lens=move(torch.tensor(lengths, dtype=torch.int32)), kv=kv, k_scale=move(scales[0]), v_scale=move(scales[1]),
                scale=1.0 / math.sqrt(size), most=max(list(lengths) + [0]), new=list(new), lengths=list(lengths), block=block)


def dequantised(cache, kv, scale):
    return cache.double() if kv == "auto" else cache.contiguous().view(FP8[kv]).double() * scale.double()


def attention_in_64_bits(case, window=None, sinks=0):
    """(out, bound) [tokens, heads, size]: the definition, and how far a result may be from it by what is rounded:

    - the result to its type: eps / 2 of its value;
    - the weights to the queries' type before they multiply V, with a sum that takes them as rounded: eps / 2 of
      sum p |v| and of the value, and half the smallest step of the type for each key (weights are at most 1, their sum
      at least 1), none of both for fp32;
    - the scores in 32 bits: head_size + 4 steps of 2^-24 of scale * sum |q k|, and a product with log2 e and a
      difference of at most three times the largest score; a weight moves by that much, relative;
    - the sums over the keys in 32 bits: a step of 2^-24 for each key, and a few for the factors."""
    query, dtype = case["query"], case["query"].dtype
    tokens, heads, size = query.shape
    out = torch.zeros(tokens, heads, size, dtype=torch.float64, device=query.device)
    bound = torch.zeros_like(out)
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    step = 0.0 if dtype == torch.float32 else torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    last = torch.finfo(dtype).eps / 2
    capacity = case["table"].size(1) * case["block"]
    group = heads // case["key"].size(2)
    first = 0
    for b, n in enumerate(case["new"]):
        length = max(0, min(int(case["seq_lens"][b]), capacity))
        j = torch.arange(length, device=query.device)
        page = case["table"][b].long()[j // case["block"]]
        there = (page >= 0) & (page < case["key"].size(0))
        key = dequantised(case["key"][page.clamp(0, case["key"].size(0) - 1), j % case["block"]], case["kv"], case["k_scale"])
        value = dequantised(case["value"][page.clamp(0, case["key"].size(0) - 1), j % case["block"]], case["kv"], case["v_scale"])
        for i in range(n):
            p = length - n + i
            seen = there & (j <= p)
            if window is not None:
                seen &= (j > p - window) | (j < sinks)
            if not bool(seen.any()):
                bound[first + i] = 1e-300
                continue
            k, v = key[seen], value[seen]
            for h in range(heads):
                q = query[first + i, h].double()
                s = (k[:, h // group] @ q) * case["scale"]
                w = torch.softmax(s, 0)
                o = w @ v[:, h // group]
                spread = w @ v[:, h // group].abs()
                terms = (k[:, h // group].abs() @ q.abs()).max() * abs(case["scale"])   # |scale| sum |q k| bounds every partial sum
                fine = 2.0 ** -24 * (2 * (size + 4) * terms + 6 * s.abs().max() + 2 * s.numel() + 32)
                out[first + i, h] = o
                bound[first + i, h] = last * o.abs() + half * (spread + o.abs()) + fine * (spread + o.abs()) + \
                    step * s.numel() * v[:, h // group].abs().amax(0) + 1e-30
        first += n
    return out, bound * 1.0001


def assert_attention(got, want, bound, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    if bool(bad.any()):
        at = bad.nonzero()[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {at}: got {got[tuple(at)].item()} want "
                             f"{want[tuple(at)].item()} bound {bound[tuple(at)].item():.3g}; worst ratio {float((off / bound).nan_to_num(9e9).max()):.3g}")


# ---- verification ----------------------------------------------------------------------------------------------------
def verify_in_64_bits(logits, row_start, drafts, accept, sample, temperatures=None):
    """The definition, one number after another: (tokens, counts)."""
    x_all = logits.detach().cpu().double().numpy()
    start, drafts = row_start.tolist(), drafts.cpu().numpy()
    accept, sample = accept.cpu().double().numpy(), sample.cpu().double().numpy()
    batch, most = drafts.shape
    t_all = np.ones(batch) if temperatures is None else temperatures.cpu().double().numpy()
    tokens, counts = np.full((batch, most + 1), -1, dtype=np.int64), np.zeros(batch, dtype=np.int64)
    for b in range(batch):
        first, end = start[b], min(start[b + 1], x_all.shape[0])
        if first < 0 or end <= first:
            continue
        n, t = min(most, end - first - 1), t_all[b]
        for k in range(n + 1):
            x = x_all[first + k]
            nan = np.isnan(x)
            best = int(np.argmax(nan)) if nan.any() else int(np.argmax(x))
            draft = int(drafts[b, k]) if k < n else -1
            known = 0 <= draft < x.size
            spread = t > 0 and np.isfinite(x[best])
            if spread:
                with np.errstate(invalid="ignore"):
                    w = np.where(x == -np.inf, 0.0, np.exp((x - x[best]) * (1.0 / t)))
            if k < n and known and np.isfinite(x[best]):
                if (accept[b, k] * w.sum() < w[draft]) if spread else draft == best:
                    tokens[b, k] = draft
                    continue
            token = best
            if spread:
                if known:
                    w[draft] = 0.0
                sums = np.cumsum(w)
                over = (sums > sample[b] * sums[-1]) & (w > 0)
                if over.any():
                    token = int(np.argmax(over))
                elif (w > 0).any():
                    token = int(np.nonzero(w > 0)[0][-1])
            tokens[b, k] = token
            counts[b] = k + 1
            break
    return torch.from_numpy(tokens), torch.from_numpy(counts)
