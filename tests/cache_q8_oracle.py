"""The 8-bit cache in 64 bits, for the tests: codes, scales, attention over them, and how far a kernel's result may be off."""

from __future__ import annotations

import math

import torch


def quantise(x: torch.Tensor):
    """Codes (int8) and scales (float32) of rows x [..., D]: the nearest multiples of a / 127, of two equally near ones the even."""
    rows = x.double()
    a = rows.abs().amax(-1)
    bad = ~torch.isfinite(a)
    safe = torch.where((a > 0) & ~bad, a, 1.0)
    codes = torch.round(torch.where(bad[..., None], 0.0, rows) * 127 / safe[..., None])
    codes = torch.where(bad[..., None], 0.0, codes).to(torch.int8)
    scales = torch.where(bad, math.nan, a / 127).float()
    return codes, scales


def pages_case(heads, kv_heads, dim, page, q_lens, ctx_lens, dtype, seed=0, device="cpu", q_scale=1.0):
    """Sequences scattered over shuffled pages.  Places behind a sequence's last key, pages that nobody holds and what lies
    behind a table row's last page hold codes of any kind and NaN scales."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-c // page) for c in ctx_lens]
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=g).tolist()
    codes = [torch.randint(-128, 128, (pages, page, kv_heads, dim), generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [torch.full((pages, kv_heads, page), math.nan) for _ in range(2)]
    width = max(max(held), 1) + 2
    table = torch.full((len(ctx_lens), width), -1, dtype=torch.int32)
    sequences = []
    for s, context in enumerate(ctx_lens):
        mine = [order.pop() for _ in range(held[s])]
        table[s, : held[s]] = torch.tensor(mine, dtype=torch.int32)
        pair = []
        for kind in range(2):
            x = torch.randn(context, kv_heads, dim, generator=g)
            x = x * torch.where(torch.rand(kv_heads, dim, generator=g) < 0.05, 6.0, 1.0)
            c, sc = quantise(x)
            for j in range(context):
                codes[kind][mine[j // page], j % page] = c[j]
                scales[kind][mine[j // page], :, j % page] = sc[j]
            pair.append((c, sc))
        sequences.append(pair)
    tokens = sum(q_lens)
    starts = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32)
    q = (torch.randn(tokens, heads * dim, generator=g) * q_scale).to(dtype)
    owner = torch.repeat_interleave(torch.arange(len(q_lens)), torch.tensor(q_lens)).to(torch.int32)
    case = dict(codes_k=codes[0], codes_v=codes[1], scales_k=scales[0], scales_v=scales[1], table=table, q=q, q_start=starts,
                ctx_len=torch.tensor(ctx_lens, dtype=torch.int32), seq_of=owner)
    case = {k: v.to(device) for k, v in case.items()}
    case["sequences"] = [[(c.to(device), sc.to(device)) for c, sc in pair] for pair in sequences]
    return case


def attention(q, sequences, q_lens, ctx_lens, heads, kv_heads, dim, scale, window=None, chunk=None):
    """(outputs [tokens, heads * dim] in 64 bits, how far a kernel may be off them).

    The bound counts, with u = 2^-23 for an addition in a product's 32-bit sums (which may round toward zero):
      a score: dim / 16 additions of products, their factors and, for 32-bit queries, what two 11-bit parts leave (2^-22), all
               relative to sum |q k|; the subtraction of the base and the exponential, 2^-22 each of the argument's size
      a weight: half a step of float16 (2^-11), or of two parts of it (2^-22) for 32-bit queries, and never less than half of
                float16's least step, 2^-25, where a weight of one at the largest value scale seen stands at 2^8 or more (and the
                sums hold the largest score's exponential, one, or up to 2^6 where the base lags): 2^-33 of that scale a key,
                times codes of up to 127
      a sum over n keys: n / 16 additions and as many rescalings
    all relative to sum p |v| / sum p, and half a step of the output's type relative to the output."""
    u = 2.0 ** -23
    wide = q.dtype == torch.float32
    half_step = 2.0 ** -24 if wide else 2.0 ** -8
    outs, bounds, at = [], [], 0
    group = heads // kv_heads
    for (keys, values), new, context in zip(sequences, q_lens, ctx_lens):
        k = keys[0].double() * keys[1].double()[..., None]
        v = values[0].double() * values[1].double()[..., None]
        rows = q[at: at + new].double().view(new, heads, dim)
        at += new
        position = torch.arange(context - new, context, device=q.device)
        key = torch.arange(context, device=q.device)
        seen = key <= position[:, None]
        if window:
            seen &= key > position[:, None] - window
        if chunk:
            seen &= key // chunk == position[:, None] // chunk
        out, bound = torch.zeros(new, heads, dim, dtype=torch.float64, device=q.device), torch.zeros(new, heads, dim, dtype=torch.float64, device=q.device)
        some = seen.any(-1)
        for head in range(heads if context else 0):
            g = head // group
            z = (rows[:, head] @ k[:, g].T) * scale
            size = (rows[:, head].abs() @ k[:, g].abs().T) * abs(scale)
            p = torch.softmax(torch.where(seen, z, -math.inf), -1)
            p = torch.where(seen & some[:, None], p, 0.0)   # a row that sees nothing is zeros
            # a key that is not seen has no part in it, whatever it holds
            vv = torch.where(seen.any(0)[:, None], v[:, g], 0.0)
            out[:, head] = p @ vv
            there = torch.where(seen, size, 0.0).amax(-1, keepdim=True)
            score = there * ((dim / 16 + 4) * u + (2.0 ** -22 if wide else 0.0)) + 2.0 ** -21 * (there + 32)
            sums = (context / 8 + 16) * u
            least = seen.sum(-1, keepdim=True) * 2.0 ** -33 * 127 * torch.where(seen, values[1][:, g].double(), 0.0).amax(-1, keepdim=True)
            bound[:, head] = least + (p @ vv.abs()) * (2 * score + (2.0 ** -22 if wide else 2.0 ** -11) + 2 * sums)
        outs.append(out.view(new, heads * dim))
        bounds.append((bound + half_step * out.abs()).view(new, heads * dim))
    return torch.cat(outs), torch.cat(bounds)
