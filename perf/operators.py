"""The 8-bit cache's operators, each by its plain form and by the framework's kernels.

A cache page holds `page` tokens: int8 codes [pages, page, kv heads, head size] and one float32 scale per token and kv head,
[pages, kv heads, page], for the keys and again for the values.  The fields of a case:

  kind     "store":  `tokens` new keys and values are quantised into their pages and read back from there
           "read":   `tokens` keys and values are read back
           "attend": `portions` sequences bring up to `tokens` new tokens each and `singles` sequences one each; every
                     sequence's context, new tokens included, is up to `context` keys long
  heads, kv_heads, dim, page, dtype; window: a query sees that many latest keys (0: all)
"""

import functools
import math

import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
HEADS = [(14, 2), (12, 2), (28, 4), (40, 8), (16, 2), (6, 3), (4, 2), (64, 8)]   # the package's shapes and the tests'


def store(name, tokens, kv_heads, dim, page=16, dtype="bfloat16", kind="store"):
    given = {"kind": kind, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}
    return given if name is None else {"name": name, **given}


def attend(name, heads, kv_heads, dim, portions=0, tokens=0, singles=0, context=0, page=16, dtype="bfloat16", window=0):
    given = {"kind": "attend", "heads": heads, "kv_heads": kv_heads, "dim": dim, "portions": portions, "tokens": tokens,
             "singles": singles, "context": context, "page": page, "dtype": dtype, "window": window}
    return given if name is None else {"name": name, **given}


def listed():
    return [
        # one user decoding at 7B widths: one token's keys and values, latency alone
        store("store_7b_1", 1, 4, 128),
        # a long prompt at 7B widths, in one step
        store("store_7b_2048", 2048, 4, 128),
        # the 32-bit path at the tests' sizes, a ragged count
        store("store_fp32_1037", 1037, 3, 32, page=8, dtype="float32"),
        # a request's cache handed out: 14B widths, a long context
        store("read_14b_32768", 32768, 8, 128, kind="read"),
        # one user in the middle of an answer at 7B widths: latency
        attend("decode_7b_b1", 28, 4, 128, singles=1, context=517),
        # the headline's batch of eight at about 1,024 tokens
        attend("decode_7b_b8", 28, 4, 128, singles=8, context=1024),
        # many users at 14B widths, what an 8-bit cache makes room for
        attend("decode_14b_b64", 40, 8, 128, singles=64, context=4096),
        # one long document at 14B widths
        attend("decode_14b_long", 40, 8, 128, singles=1, context=65521),
        # the headline's long prompt, whole
        attend("prompt_7b_2048", 28, 4, 128, portions=1, tokens=2048, context=2048),
        # a portion under the stock token budget, late in a long document
        attend("chunk_14b_512", 40, 8, 128, portions=1, tokens=512, context=8192),
        # a step of the mixed workload at 1.5B widths: a portion beside decoding requests
        attend("mixed_1.5b", 12, 2, 128, portions=1, tokens=475, singles=37, context=1115),
        # the 32-bit path at the tests' sizes: prompts of uneven lengths
        attend("prompts_fp32", 6, 3, 32, portions=5, tokens=70, context=150, page=8, dtype="float32"),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    page = rng.choice([8, 16, 16, 32, 64])
    heads, kv_heads = rng.choice(HEADS)
    dim = rng.choice([32, 64, 64, 128, 128, 128])
    kind = rng.choice(["store", "read", "attend", "attend", "attend", "attend"])
    if kind != "attend":
        return store(None, _log(rng, 1, 30000 if kind == "read" else 5000), kv_heads, dim, page, dtype, kind)
    window = _log(rng, 5, 2000) if rng.random() < 0.25 else 0
    if rng.random() < 0.5:
        singles = _log(rng, 1, 80)
        return attend(None, heads, kv_heads, dim, singles=singles, context=_log(rng, 1, min(60000, 200000 // singles)), page=page,
                      dtype=dtype, window=window)
    portions, singles = rng.choice([1, 1, 2, 3]), rng.choice([0, 0, 1, 9])
    # the plain form pads every sequence to the longest portion and context: as many scores as the largest listed case has
    room = 1.6e8 / (heads * (portions + singles))
    tokens = _log(rng, 2, min(400 if dtype == "float32" else 2000, int(room ** 0.5)))
    context = tokens + _log(rng, 1, max(1, min(9000, int(room / tokens) - tokens))) - 1
    return attend(None, heads, kv_heads, dim, portions, tokens, singles, context, page, dtype, window)


def _lengths(case):
    """Every sequence's (new tokens, context): uneven, the first of each sort as long as the case says."""
    entries = []
    for i in range(case["portions"]):
        new = max(1, case["tokens"] - i * case["tokens"] * 5 // 16)
        before = case["context"] - case["tokens"]
        entries.append((new, new + before - i * before * 3 // 16))
    for i in range(case["singles"]):
        entries.append((1, max(1, case["context"] - case["context"] * ((i * 7) % 16) // 32 - (i % 5 if case["context"] > 64 else 0))))
    return entries


def _visible(new, context, window):
    """Pairs of a query and a key that it sees."""
    if not window:
        return new * context - new * (new - 1) // 2
    return sum(min(window, context - new + t + 1) for t in range(new))


def _seen(new, context, window):
    """Keys that any query of the sequence sees."""
    return context if not window else min(context, new + window - 1)


def work(case):
    e, width = TYPES[case["dtype"]].itemsize, case["kv_heads"] * case["dim"]
    if case["kind"] != "attend":
        rows = 2 * case["tokens"]
        plain, coded = rows * width * e, rows * (width + 4 * case["kv_heads"])
        return {"bytes": plain + coded + (plain if case["kind"] == "store" else 0), "flops": 3 * rows * width}
    entries, q_width = _lengths(case), case["heads"] * case["dim"]
    rows = 2 * sum(n for n, _ in entries) * q_width * e
    coded = 2 * sum(_seen(n, c, case["window"]) for n, c in entries) * (width + 4 * case["kv_heads"])
    return {"bytes": rows + coded, "flops": 4 * q_width * sum(_visible(n, c, case["window"]) for n, c in entries)}


def _rows(g, count, kv_heads, dim):
    """Projected keys as they come: normal, a few channels several times as large."""
    x = torch.randn(count, kv_heads, dim, generator=g, device="cuda")
    loud = torch.rand(kv_heads, dim, generator=g, device="cuda") < 0.05
    return x * torch.where(loud, 6.0, 1.0)


def _page_pool(g, pages, case):
    """Codes and scales of whole pages; what no sequence has written holds anything."""
    kv_heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    x = _rows(g, pages * page, kv_heads, dim)
    largest = x.abs().amax(-1)
    codes = torch.round(x * 127 / largest[..., None]).to(torch.int8).view(pages, page, kv_heads, dim)
    return codes, (largest / 127).view(pages, page, kv_heads).transpose(1, 2).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kv_heads, dim, page = TYPES[case["dtype"]], case["kv_heads"], case["dim"], case["page"]
    if case["kind"] != "attend":
        n = case["tokens"]
        pages = -(-n // page) + 3
        slots = (torch.randperm(pages, generator=g, device="cuda")[:, None] * page + torch.arange(page, device="cuda")).view(-1)
        slots = slots[:n].to(torch.int32)
        codes_k, scales_k = _page_pool(g, pages, case)
        codes_v, scales_v = _page_pool(g, pages, case)
        state = {"case": case, "codes_k": codes_k, "scales_k": scales_k, "codes_v": codes_v, "scales_v": scales_v, "slots": slots,
                 "k_out": torch.empty(n, kv_heads * dim, dtype=dtype, device="cuda"),
                 "v_out": torch.empty(n, kv_heads * dim, dtype=dtype, device="cuda")}
        if case["kind"] == "store":
            state["k"] = _rows(g, n, kv_heads, dim).view(n, -1).to(dtype)
            state["v"] = _rows(g, n, kv_heads, dim).view(n, -1).to(dtype)
        return state
    entries = _lengths(case)
    new, contexts = [n for n, _ in entries], [c for _, c in entries]
    held = [-(-c // page) for c in contexts]
    pages = sum(held) + 5
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    width = max(held)
    column = torch.arange(width, device="cuda")
    held_t = torch.tensor(held, device="cuda")
    first = torch.cumsum(held_t, 0) - held_t
    mine = column < held_t[:, None]
    table = torch.where(mine, order[torch.where(mine, first[:, None] + column, 0)], -1).to(torch.int32)
    codes_k, scales_k = _page_pool(g, pages, case)
    codes_v, scales_v = _page_pool(g, pages, case)
    contexts_t = torch.tensor(contexts, device="cuda")
    # places behind a sequence's last key, and pages that nobody holds, keep what an earlier request left, or nothing at all
    key = column[:, None] * page + torch.arange(page, device="cuda")
    written = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    written[table[mine].long()] = (key[None] < contexts_t[:, None, None])[mine]
    for scales in (scales_k, scales_v):
        scales.masked_fill_(~written[:, None, :], float("nan"))
    tokens = sum(new)
    new_t = torch.tensor(new, device="cuda")
    q = torch.randn(tokens, case["heads"], dim, generator=g, device="cuda") * 1.3
    return {"case": case, "codes_k": codes_k, "scales_k": scales_k, "codes_v": codes_v, "scales_v": scales_v,
            "q": q.view(tokens, -1).to(dtype), "block_table": table,
            "q_start": torch.cat([new_t.new_zeros(1), torch.cumsum(new_t, 0)]).to(torch.int32), "ctx_len": contexts_t.to(torch.int32),
            "seq_of_token": torch.repeat_interleave(torch.arange(len(new), device="cuda"), new_t, output_size=tokens).to(torch.int32),
            "out": torch.empty(tokens, case["heads"] * dim, dtype=dtype, device="cuda"), "q_lens": new, "max_ctx_len": max(contexts)}


@functools.lru_cache(maxsize=None)
def _kernels(dtype):
    from shrike_b200.ops.cuda_ops import CudaOps

    return CudaOps(TYPES[dtype])


def _own(state):
    from shrike_b200.cache.quantised import QuantisedPages

    case = state["case"]
    ops = _kernels(case["dtype"])
    keys, values = QuantisedPages(state["codes_k"], state["scales_k"]), QuantisedPages(state["codes_v"], state["scales_v"])
    if case["kind"] == "attend":
        ops.paged_attention(
            state["q"], keys, values, state["block_table"], state["q_start"], state["ctx_len"], state["seq_of_token"], case["heads"],
            case["kv_heads"], case["dim"], case["dim"] ** -0.5, case["window"] or None, state["out"], max_q_len=max(state["q_lens"]),
            max_ctx_len=state["max_ctx_len"], min_q_len=min(state["q_lens"]), q_lens=state["q_lens"])
        return state["out"]
    if case["kind"] == "store":
        ops.kv_write(state["k"], state["v"], keys, values, state["slots"])
    ops.kv_read(keys, values, state["slots"], state["k_out"], state["v_out"])
    return state["k_out"], state["v_out"]


def _write(x, codes, scales, slots):
    """In 64 bits: half a step is a border of the rounding, and x = a / 2 lies on one."""
    page, kv_heads, dim = codes.shape[1:]
    x = x.view(-1, kv_heads, dim).double()
    largest = x.abs().amax(-1)
    coded = torch.round(x * 127 / torch.where(largest > 0, largest, 1.0)[..., None])
    codes.view(-1, kv_heads, dim)[slots] = coded.to(torch.int8)
    scales[slots // page, :, slots % page] = (largest / 127).float()


def _read(codes, scales, slots, out):
    page, kv_heads, dim = codes.shape[1:]
    x = codes.view(-1, kv_heads, dim)[slots].float() * scales[slots // page, :, slots % page][..., None]
    return out.copy_(x.view(out.shape))


def _in_order(codes, scales, table, contexts):
    """float32 [sequences, kv heads, keys, head size] from the pages, zeros where a sequence has no key."""
    sequences, blocks = table.shape
    page, kv_heads, dim = codes.shape[1:]
    at = table.clamp(min=0).long()
    x = codes[at].float() * scales[at].transpose(2, 3)[..., None]
    x = x.view(sequences, blocks * page, kv_heads, dim).transpose(1, 2)
    here = torch.arange(blocks * page, device=x.device) < contexts[:, None]
    return torch.where(here[:, None, :, None], x, 0.0)


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["kind"] != "attend":
        slots = state["slots"].long()
        if case["kind"] == "store":
            _write(state["k"], state["codes_k"], state["scales_k"], slots)
            _write(state["v"], state["codes_v"], state["scales_v"], slots)
        return (_read(state["codes_k"], state["scales_k"], slots, state["k_out"]),
                _read(state["codes_v"], state["scales_v"], slots, state["v_out"]))
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group, q, contexts = heads // kv_heads, state["q"], state["ctx_len"].long()
    starts, owner = state["q_start"].long(), state["seq_of_token"].long()
    keys = _in_order(state["codes_k"], state["scales_k"], state["block_table"], contexts)
    values = _in_order(state["codes_v"], state["scales_v"], state["block_table"], contexts)
    sequences, longest = len(contexts), max(state["q_lens"])
    place = torch.arange(q.shape[0], device=q.device) - starts[owner]
    rows = q.new_zeros(sequences, longest, kv_heads, group, dim, dtype=torch.float32)
    rows[owner, place] = q.float().view(-1, kv_heads, group, dim)
    rows = rows.permute(0, 2, 3, 1, 4).reshape(sequences, kv_heads, group * longest, dim)
    scores = torch.matmul(rows, keys.transpose(2, 3)).view(sequences, kv_heads, group, longest, -1).mul_(dim ** -0.5)
    last = (contexts - (starts[1:] - starts[:-1]))[:, None] + torch.arange(longest, device=q.device)   # a query's own position
    key = torch.arange(scores.shape[-1], device=q.device)
    hidden = (key > last[..., None]) | (key >= contexts[:, None, None])
    if case["window"]:
        hidden |= key <= last[..., None] - case["window"]
    hidden &= (last < contexts[:, None])[..., None]   # a padding row may see anything: it is dropped below
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(sequences, kv_heads, group * longest, -1), values).view(sequences, kv_heads, group, longest, dim) / total
    out = out.permute(0, 3, 1, 2, 4)[owner, place]
    return state["out"].copy_(out.reshape(state["out"].shape))


def exact(case, seed):
    state = prepare(case, seed)
    kv_heads, dim, page = case["kv_heads"], case["dim"], case["page"]

    def value(codes, scales, slots):
        slots = slots.long()
        return codes.view(-1, kv_heads, dim)[slots].double() * scales.double().transpose(1, 2).reshape(-1, kv_heads, 1)[slots]

    if case["kind"] == "read":
        return tuple(value(state["codes_" + x], state["scales_" + x], state["slots"]).view(case["tokens"], -1) for x in "kv")
    if case["kind"] == "store":
        found = []
        for x in "kv":
            rows = state[x].double().view(-1, kv_heads, dim)
            step = rows.abs().max(-1, keepdim=True).values / 127
            # the nearest multiple of the step; of two equally near ones the even one
            found.append((torch.where(step > 0, (rows * 127 / (step * 127)).round(), 0.0) * step).view(case["tokens"], -1))
        return tuple(found)
    outs, at = [], 0
    for index, (new, context) in enumerate(_lengths(case)):
        key = torch.arange(context, device="cuda")
        slots = state["block_table"][index].long()[key // page] * page + key % page
        keys, values = value(state["codes_k"], state["scales_k"], slots), value(state["codes_v"], state["scales_v"], slots)
        q = state["q"][at: at + new].double().view(new, case["heads"], dim)
        position = torch.arange(context - new, context, device="cuda")
        seen = key <= position[:, None]
        if case["window"]:
            seen &= key > position[:, None] - case["window"]
        heads = []
        for head in range(case["heads"]):
            g = head // (case["heads"] // kv_heads)
            score = (q[:, head] @ keys[:, g].T) / math.sqrt(dim)
            heads.append(torch.softmax(torch.where(seen, score, -math.inf), -1) @ values[:, g])
        outs.append(torch.stack(heads, 1).view(new, -1))
        at += new
    return torch.cat(outs)
