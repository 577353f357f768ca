"""Workloads of the 8-bit paged KV cache and of the cache's page operators.

Three groups of calls:

  rows     a step's K / V rows quantised into the 8-bit cache and the
           sequences' rows read back in bf16 (what a chunked prompt's attention
           over its cached prefix takes)
  decode   attention of one new token per sequence over the 8-bit paged cache
  pages    copying, forking (shared full pages, the last one copied on write),
           freeing and compacting the pages of a cache

The 8-bit cache holds e4m3 values [num_blocks, block_size, Hk, 128] and one
exponent byte per (token, kv head) row, [num_blocks, Hk, block_size]: a row
reads as e4m3 * 2^(byte - 127).
"""

import math
import os
import random
import sys

import torch

own = False

HEAD_DIM = 128


# where this repository's package lies (it is imported only for its own calls)
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nanokv-llm_b200"))


# ---------------------------------------------------------------- cases
def listed():
    return [
        # One chat of a 16-head / 8-kv-head model, right after a short prompt: all latency.
        {"name": "decode_one_chat", "op": "decode", "batch": 1, "q_heads": 16, "kv_heads": 8, "block": 256,
         "min_len": 700, "max_len": 700, "empty": 0},
        # A serving batch of the 32-head / 8-kv-head model with ragged contexts and graph-padding rows.
        {"name": "decode_batch_ragged", "op": "decode", "batch": 61, "q_heads": 32, "kv_heads": 8, "block": 256,
         "min_len": 1, "max_len": 4000, "empty": 5},
        # Few long contexts on a quarter of the heads (tensor parallel over 4): the length is what is split.
        {"name": "decode_long_shard", "op": "decode", "batch": 4, "q_heads": 8, "kv_heads": 2, "block": 256,
         "min_len": 90001, "max_len": 131072, "empty": 0},
        # A full decode batch of long contexts: all bandwidth.
        {"name": "decode_full", "op": "decode", "batch": 128, "q_heads": 32, "kv_heads": 8, "block": 256,
         "min_len": 1000, "max_len": 8192, "empty": 0},
        # Short prompts stored and read back: the smallest prefill step.
        {"name": "rows_short_prompts", "op": "rows", "batch": 3, "kv_heads": 8, "q_heads": 16, "block": 256,
         "min_len": 1, "max_len": 150, "new_share": 1.0},
        # The next chunk of several long prompts: new rows stored, prefix and chunk read back.
        {"name": "rows_prompt_chunk", "op": "rows", "batch": 8, "kv_heads": 8, "q_heads": 32, "block": 256,
         "min_len": 2001, "max_len": 8192, "new_share": 0.5},
        # Pages duplicated one by one, K and V of every layer: a prefix copied for another owner.
        {"name": "pages_copy", "op": "copy", "layers": 28, "kv_heads": 8, "block": 256, "pages": 64, "pairs": 21},
        # Four samples of one prompt: the pages shared, the last one copied.
        {"name": "pages_fork_samples", "op": "fork", "layers": 28, "kv_heads": 2, "block": 256, "prompts": 1,
         "branches": 4, "min_len": 549, "max_len": 549, "rows": 16, "spare": 12},
        # Three branches for each of many prompts.
        {"name": "pages_fork_batch", "op": "fork", "layers": 4, "kv_heads": 8, "block": 256, "prompts": 48,
         "branches": 3, "min_len": 1, "max_len": 1500, "rows": 256, "spare": 31},
        # Branches on full pages opened and dropped again: no byte of the cache moves.
        {"name": "pages_drop_branches", "op": "drop", "layers": 1, "kv_heads": 1, "block": 16, "prompts": 16,
         "branches": 4, "min_len": 16, "max_len": 2048, "rows": 128, "spare": 100},
        # A small pool after a few requests ended.
        {"name": "pages_compact_small", "op": "compact", "layers": 28, "kv_heads": 1, "block": 256, "pages": 96,
         "live": 23, "rows": 16},
        # A big pool, half empty and scattered, brought together.
        {"name": "pages_compact_pool", "op": "compact", "layers": 4, "kv_heads": 8, "block": 256, "pages": 512,
         "live": 201, "rows": 128},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "decode", "rows", "rows", "copy", "fork", "drop", "compact"])
    block = rng.choice([16, 32, 64, 128, 256, 256, 512])
    kv_heads = rng.choice([1, 2, 4, 8])
    if op == "decode":
        group = rng.choice([1, 2, 4, 5, 8, 16])
        batch = _log_int(rng, 1, 128)
        # at most the tokens x kv heads of the largest listed batch
        high = min(131072, 128 * 4000 * 8 // (batch * kv_heads))
        high = _log_int(rng, 64, max(64, high))
        return {"op": op, "batch": batch, "q_heads": group * kv_heads, "kv_heads": kv_heads, "block": block,
                "min_len": _log_int(rng, 1, high), "max_len": high, "empty": rng.choice([0, 0, batch // 8])}
    if op == "rows":
        batch = _log_int(rng, 1, 32)
        high = _log_int(rng, 1, max(1, 30000 * 8 // (batch * kv_heads)))
        return {"op": op, "batch": batch, "kv_heads": kv_heads, "q_heads": 2 * kv_heads, "block": block,
                "min_len": _log_int(rng, 1, high), "max_len": high, "new_share": rng.choice([0.1, 0.5, 1.0])}
    layers = _log_int(rng, 1, 36)
    page = 2 * layers * block * kv_heads * HEAD_DIM * 2  # bytes of a page of all layers
    if op == "copy":
        most = min(400, (1500 << 20) // page)
        pages = _log_int(rng, 4, max(4, most))
        return {"op": op, "layers": layers, "kv_heads": kv_heads, "block": block, "pages": pages,
                "pairs": _log_int(rng, 1, max(1, min(pages // 3, (600 << 20) // page)))}
    if op in ("fork", "drop"):
        high = _log_int(rng, block, 1500)
        prompts = _log_int(rng, 1, 40)
        branches = rng.randint(1, 4)
        while prompts > 1 and prompts * (branches + 1 + high // block) * page > (1200 << 20):
            prompts //= 2
        case = {"op": op, "layers": layers, "kv_heads": kv_heads, "block": block, "prompts": prompts,
                "branches": branches, "min_len": _log_int(rng, 1, high), "max_len": high,
                "rows": prompts * (branches + 1) + rng.randint(0, 20), "spare": rng.randint(0, 20)}
        if op == "drop":
            case["min_len"] = max(case["min_len"], block)
        return case
    pages = _log_int(rng, 8, max(8, min(500, (1500 << 20) // page)))
    return {"op": op, "layers": layers, "kv_heads": kv_heads, "block": block, "pages": pages,
            "live": rng.randint(1, max(1, pages // 2)), "rows": rng.randint(1, 64)}


def _lens(case, count):
    """The case's lengths: spread over its range, the same for every seed (what a pass moves depends on them)."""
    rng = random.Random("%s/%s/%s/%s" % (count, case["min_len"], case["max_len"], case["block"]))
    lens = [rng.randint(case["min_len"], case["max_len"]) for _ in range(count)]
    if case["op"] == "drop":
        lens = [max(1, n // case["block"]) * case["block"] for n in lens]
    for i in range(case.get("empty", 0)):
        lens[(7 * i + 3) % count] = 0
    return lens


def _ceil(a, b):
    return -(-a // b)


def _new_lens(case, lens):
    """Rows of each sequence that the step brings."""
    return [max(1, int(n * case["new_share"])) for n in lens]


def work(case):
    op = case["op"]
    if op == "decode":
        tokens = sum(_lens(case, case["batch"]))
        io = 2 * case["batch"] * case["q_heads"] * HEAD_DIM * 2
        return {"bytes": tokens * case["kv_heads"] * (2 * HEAD_DIM + 2) + io,
                "flops": 4 * tokens * case["q_heads"] * HEAD_DIM}
    if op == "rows":
        lens = _lens(case, case["batch"])
        new, total = sum(_new_lens(case, lens)), sum(lens)
        row16, row8 = 4 * HEAD_DIM * case["kv_heads"], (2 * HEAD_DIM + 2) * case["kv_heads"]
        # new rows read in bf16 and written in 8 bits; the older ones read in 8 bits; all written in bf16
        return {"bytes": new * (row16 + row8) + (total - new) * row8 + total * row16,
                "flops": (new + total) * case["kv_heads"] * 2 * HEAD_DIM}
    token = 4 * HEAD_DIM * case["kv_heads"] * case["layers"]
    if op == "copy":
        return {"bytes": 2 * case["pairs"] * case["block"] * token, "flops": 0}
    if op in ("fork", "drop"):
        lens = _lens(case, case["prompts"])
        tails = sum(n % case["block"] for n in lens) * case["branches"]
        pages = sum(_ceil(n, case["block"]) for n in lens)
        entries = 4 * (pages + (1 if op == "fork" else 3) * pages * case["branches"])
        return {"bytes": 2 * tails * token + entries, "flops": 0}
    live, moves = _live(case)
    return {"bytes": 2 * moves * case["block"] * token + 8 * case["pages"] + 8 * len(live), "flops": 0}


def _live(case):
    """The live pages of a compaction and how many of them lie past the first len(live)."""
    rng = random.Random("%s/%s/%s" % (case["pages"], case["live"], case["rows"]))
    live = rng.sample(range(case["pages"]), case["live"])
    return live, sum(p >= len(live) for p in live)


# ---------------------------------------------------------------- inputs
def _pow2(byte):
    """2^(byte - 127) from an exponent byte in [1, 254], exactly."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _quantise(x):
    """Rows [..., 128] to e4m3 values and an exponent byte each."""
    v = x.float()
    top = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(-1)
    frac, exp = torch.frexp(top)  # top = frac * 2^exp, frac in [0.5, 1)
    k = exp - 9 + (frac > 0.875).to(torch.int32)  # the smallest k with top <= 448 * 2^k
    k = torch.where(top > 0, k, torch.full_like(k, -117)).clamp(-117, 119)
    q = (v * _pow2(127 - k).unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return q, (k + 127).to(torch.uint8)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(g, n, heads):
    """K or V rows as a model's projections give them: normal, with some channels larger and rows of uneven norm."""
    x = torch.randn(n, heads, HEAD_DIM, generator=g, device="cuda")
    channel = 1 + 3 * (torch.rand(heads, HEAD_DIM, generator=g, device="cuda") > 0.95).float()
    norm = torch.exp(0.4 * torch.randn(n, heads, 1, generator=g, device="cuda"))
    return (x * channel * norm).to(torch.bfloat16)


def _tables(g, lens, block, pages):
    """Block tables over a shuffled pool, -1 padded."""
    perm = torch.randperm(pages, generator=g, device="cuda").tolist()
    width, table, at = max(1, max(_ceil(n, block) for n in lens)), [], 0
    for n in lens:
        m = _ceil(n, block)
        table.append(perm[at:at + m] + [-1] * (width - m))
        at += m
    return torch.tensor(table, dtype=torch.int32, device="cuda")


def _cache8(g, pages, block, heads):
    """An 8-bit cache full of stored rows."""
    data = torch.empty(pages, block, heads, HEAD_DIM, dtype=torch.float8_e4m3fn, device="cuda")
    exps = torch.empty(pages, heads, block, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (block * heads * HEAD_DIM))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        q, e = _quantise(_rows(g, n * block, heads))
        data[at:at + n] = q.view(n, block, heads, HEAD_DIM)
        exps[at:at + n] = e.view(n, block, heads).transpose(1, 2)
    return data, exps


def _stack(g, case, pages):
    """The reference's cache of a whole model: [K / V, layer, page, token, kv head, dim] in bf16."""
    shape = (2, case["layers"], pages, case["block"], case["kv_heads"], HEAD_DIM)
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g, op, block = _gen(seed), case["op"], case["block"]
    s = {"case": case, "op": op, "block": block}
    if op == "decode":
        lens = _lens(case, case["batch"])
        pages = sum(_ceil(n, block) for n in lens) + 3
        s["k"], s["ke"] = _cache8(g, pages, block, case["kv_heads"])
        s["v"], s["ve"] = _cache8(g, pages, block, case["kv_heads"])
        s["tables"], s["lens"] = _tables(g, lens, block, pages), _ints(lens)
        s["q"] = torch.randn(case["batch"], case["q_heads"], HEAD_DIM, generator=g, device="cuda").to(torch.bfloat16)
        return s
    if op == "rows":
        lens = _lens(case, case["batch"])
        new = _new_lens(case, lens)
        pages = sum(_ceil(n, block) for n in lens) + 2
        heads, total = case["kv_heads"], sum(lens)
        s["k"], s["ke"] = _cache8(g, pages, block, heads)
        s["v"], s["ve"] = _cache8(g, pages, block, heads)
        s["tables"] = _tables(g, lens, block, pages)
        s["cu"] = _ints([sum(lens[:i]) for i in range(len(lens) + 1)])
        s["total"] = total
        # the step's slots, and the rows as the slices of a qkv projection's output that they are
        table = s["tables"].tolist()
        slots = [table[b][j // block] * block + j % block for b, n in enumerate(lens) for j in range(n - new[b], n)]
        s["slots"] = _ints(slots)
        qkv = torch.cat([_rows(g, len(slots), case["q_heads"]), _rows(g, len(slots), heads), _rows(g, len(slots), heads)], 1)
        qkv = qkv.view(len(slots), -1)
        at = case["q_heads"] * HEAD_DIM
        s["key"] = qkv[:, at:at + heads * HEAD_DIM].view(-1, heads, HEAD_DIM)
        s["value"] = qkv[:, at + heads * HEAD_DIM:].view(-1, heads, HEAD_DIM)
        return s
    if op == "copy":
        perm = torch.randperm(case["pages"], generator=g, device="cuda").to(torch.int32)
        n = case["pairs"]
        s["cache"] = _stack(g, case, case["pages"])
        s["src"], s["dst"] = perm[n:2 * n].contiguous(), perm[:n].contiguous()
        return s
    if op in ("fork", "drop"):
        lens = _lens(case, case["prompts"])
        pages = sum(_ceil(n, block) for n in lens) + case["prompts"] * case["branches"] + case["spare"]
        s["cache"] = _stack(g, case, pages)
        width = max(_ceil(n, block) for n in lens) + 1
        rows = torch.randperm(case["rows"], generator=g, device="cuda")
        prompts = rows[:case["prompts"]]
        held = _tables(g, lens, block, pages)
        s["tables"] = torch.full((case["rows"], width), -1, dtype=torch.int32, device="cuda")
        s["tables"][prompts, :held.size(1)] = held
        s["lens"] = torch.zeros(case["rows"], dtype=torch.int32, device="cuda")
        s["lens"][prompts] = _ints(lens)
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
        s["refs"][held[held >= 0].long()] = 1
        s["src"] = prompts.repeat_interleave(case["branches"]).to(torch.int32)
        s["dst"] = rows[case["prompts"]:case["prompts"] * (case["branches"] + 1)].to(torch.int32)
        return s
    live, _ = _live(case)
    rows = case["rows"]
    s["cache"] = _stack(g, case, case["pages"])
    order = torch.randperm(len(live), generator=g, device="cuda").tolist()
    width = _ceil(len(live), rows) + 1
    table = [[-1] * width for _ in range(rows)]
    for i, at in enumerate(order):
        table[i % rows][i // rows] = live[at]
    s["tables"] = _ints(table)
    s["refs"] = torch.zeros(case["pages"], dtype=torch.int32, device="cuda")
    s["refs"][torch.tensor(live, device="cuda")] = 1
    if rows > 1 and table[0][0] >= 0:  # one page that two sequences share
        s["tables"][rows - 1, width - 1] = table[0][0]
        s["refs"][table[0][0]] += 1
    return s


# ---------------------------------------------------------------- plain forms
def _gather(data, exps, tables, width):
    """The sequences' rows in 32 bits, [batch, width * block, heads, 128]; unused table entries read page 0."""
    at = tables[:, :width].clamp_min(0).long()
    x = data[at].float() * _pow2(exps[at]).transpose(2, 3).unsqueeze(-1)
    return x.flatten(1, 2)


def _plain_decode(s):
    batch, q_heads, dim = s["q"].shape
    heads = s["k"].size(2)
    width = s["tables"].size(1)
    k = _gather(s["k"], s["ke"], s["tables"], width)
    q = s["q"].float().view(batch, heads, q_heads // heads, dim)
    score = torch.einsum("bhgd,bthd->bhgt", q, k) * dim ** -0.5
    del k
    masked = torch.arange(score.size(-1), device="cuda") >= s["lens"].view(-1, 1, 1, 1)
    score = score.masked_fill(masked, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    out = torch.einsum("bhgt,bthd->bhgd", p, _gather(s["v"], s["ve"], s["tables"], width))
    return out.reshape(batch, q_heads, dim).to(torch.bfloat16)


def _plain_rows(s):
    slots, block = s["slots"].long(), s["block"]
    out = []
    # where row r of the packed sequences lies in the cache
    r = torch.arange(s["total"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["cu"], r, right=True) - 1
    pos = r.long() - s["cu"].long()[seq]
    page, off = s["tables"].long()[seq, pos // block], pos % block
    for rows, data, exps in ((s["key"], s["k"], s["ke"]), (s["value"], s["v"], s["ve"])):
        q, e = _quantise(rows)
        data.view(torch.uint8)[slots // block, slots % block] = q.view(torch.uint8)
        exps[slots // block, :, slots % block] = e
        x = data.view(torch.uint8)[page, off].view(torch.float8_e4m3fn).float()
        out.append((x * _pow2(exps[page, :, off]).unsqueeze(-1)).to(torch.bfloat16))
    return out


def _plain_release(s, rows):
    """The rows' pages lose a reference; the rows are empty afterwards."""
    held = s["tables"][rows]
    used = (held >= 0).to(torch.int32)
    s["refs"].index_add_(0, held.clamp_min(0).flatten().long(), -used.flatten())
    s["tables"][rows] = -1
    s["lens"][rows] = 0


def _plain_fork(s):
    src, dst, block = s["src"].long(), s["dst"].long(), s["block"]
    _plain_release(s, dst)
    n = s["lens"][src]
    full, tail = n // block, n % block
    held = s["tables"][src]
    col = torch.arange(held.size(1), device="cuda")
    shared = col < full.unsqueeze(1)
    s["refs"].index_add_(0, held.clamp_min(0).flatten().long(), shared.flatten().to(torch.int32))
    # the i-th fork with a partial page takes the i-th lowest free page
    free = torch.argsort((s["refs"] > 0).to(torch.int32), stable=True)
    wants = tail > 0
    rank = wants.to(torch.int64).cumsum(0) - 1
    new = torch.where(wants, free[rank.clamp_min(0)], torch.full_like(rank, -1))
    last = col == full.unsqueeze(1)
    table = torch.where(shared, held, torch.full_like(held, -1))
    s["tables"][dst] = torch.where(last & wants.unsqueeze(1), new.unsqueeze(1).to(torch.int32), table)
    s["lens"][dst] = n
    s["refs"].index_add_(0, new.clamp_min(0), wants.to(torch.int32))
    # the last page's tokens; a fork without one writes its source's first page onto itself
    at = held.gather(1, torch.where(wants, full, torch.zeros_like(full)).long().unsqueeze(1)).squeeze(1).long()
    to = torch.where(wants, new, at)
    token = torch.arange(block, device="cuda")
    keep = (token < tail.unsqueeze(1)).view(1, 1, -1, block, 1, 1)
    cache = s["cache"]
    cache[:, :, to] = torch.where(keep, cache[:, :, at], cache[:, :, to])
    return new.to(torch.int32)


def _plain_compact(s):
    refs, tables, cache = s["refs"], s["tables"], s["cache"]
    pages = refs.numel()
    live = refs > 0
    count = live.sum()
    page = torch.arange(pages, device="cuda")
    # the i-th live page past the first `count` goes to the i-th free one among them
    hole = ~live & (page < count)
    mover = live & (page >= count)
    holes = torch.argsort((~hole).to(torch.int32), stable=True)
    to = torch.where(mover, holes[(mover.long().cumsum(0) - 1).clamp_min(0)], page)
    new_refs = torch.zeros_like(refs).index_add_(0, to, torch.where(live, refs, torch.zeros_like(refs)))
    new_tables = torch.where(tables >= 0, to[tables.clamp_min(0).long()].to(torch.int32), tables)
    moved = mover.nonzero().squeeze(1)
    cache[:, :, to[moved]] = cache[:, :, moved]
    return new_tables, new_refs, count.to(torch.int32).view(1)


# ---------------------------------------------------------------- one pass
def run(state):
    s, op = state, state["op"]
    if own:
        from nanokv_b200 import ops

        if op == "decode":
            return ops.paged_decode_fp8(s["q"], s["k"], s["v"], s["ke"], s["ve"], s["tables"], s["lens"], HEAD_DIM ** -0.5)
        if op == "rows":
            ops.store_kvcache_fp8(s["key"], s["value"], s["k"], s["v"], s["ke"], s["ve"], s["slots"])
            return ops.load_kvcache_fp8(s["k"], s["v"], s["ke"], s["ve"], s["tables"], s["cu"], s["total"])
        if op == "copy":
            ops.copy_pages([s["cache"]], s["src"], s["dst"], page_dim=2)
            return s["cache"]
        if op == "fork":
            new = ops.fork_pages([s["cache"]], s["tables"], s["lens"], s["refs"], s["src"], s["dst"], s["block"], page_dim=2)
            return s["cache"], s["tables"], s["lens"], s["refs"], new
        if op == "drop":
            new = ops.fork_pages([s["cache"]], s["tables"], s["lens"], s["refs"], s["src"], s["dst"], s["block"], page_dim=2)
            ops.free_pages(s["tables"], s["lens"], s["refs"], s["dst"], s["block"])
            return s["tables"], s["lens"], s["refs"], new
        tables, refs = torch.empty_like(s["tables"]), torch.empty_like(s["refs"])
        live = ops.compact_pages([s["cache"]], s["tables"], s["refs"], page_dim=2, out_block_tables=tables, out_ref_counts=refs)
        return s["cache"], tables, refs, live
    if op == "decode":
        return _plain_decode(s)
    if op == "rows":
        return _plain_rows(s)
    if op == "copy":
        s["cache"][:, :, s["dst"].long()] = s["cache"][:, :, s["src"].long()]
        return s["cache"]
    if op == "fork":
        new = _plain_fork(s)
        return s["cache"], s["tables"], s["lens"], s["refs"], new
    if op == "drop":
        new = _plain_fork(s)
        _plain_release(s, s["dst"].long())
        return s["tables"], s["lens"], s["refs"], new
    return (s["cache"], *_plain_compact(s))


# ---------------------------------------------------------------- from the definition, in 64 bits
def _two(k):
    """2^k in 64 bits from its exponent field (a power function may miss it by a last place, and with it a tie)."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _value8(bits):
    """The number an e4m3 byte stands for: sign, 4 exponent bits biased by 7, 3 fraction bits."""
    b = torch.arange(256, dtype=torch.float64, device="cuda")
    mag = b % 128
    e, m = torch.floor(mag / 8), mag % 8
    x = torch.where(e > 0, (8 + m) * _two(e - 10), m * _two(e * 0 - 9))
    x = torch.where(mag == 127, torch.full_like(x, math.nan), x)
    return torch.where(b >= 128, -x, x)[bits.long()]


def _exact_decode(s):
    q = s["q"].double()
    batch, q_heads, dim = q.shape
    heads, block = s["k"].size(2), s["block"]
    group, out = q_heads // heads, []
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            out.append(torch.zeros(q_heads, dim, dtype=torch.float64, device="cuda"))
            continue
        pages = s["tables"][b, :_ceil(n, block)].long()
        rows = []
        for h in range(heads):
            both = []
            for data, exps in ((s["k"], s["ke"]), (s["v"], s["ve"])):
                x = _value8(data.view(torch.uint8)[pages, :, h].reshape(-1, dim)[:n])
                both.append(x * _two(exps[pages, h].reshape(-1)[:n].long() - 127).unsqueeze(1))
            k, v = both
            rows.append(torch.softmax(q[b, h * group:(h + 1) * group] @ k.T / math.sqrt(dim), -1) @ v)
        out.append(torch.cat(rows))
    return torch.stack(out)


def _exact_rows(s):
    """Each row rounded to the nearest of its 8-bit numbers, by search among them."""
    grid = _value8(torch.arange(127, device="cuda"))
    block, out = s["block"], []
    cu, table = s["cu"].tolist(), s["tables"]
    for rows, data, exps in ((s["key"], s["k"], s["ke"]), (s["value"], s["v"], s["ve"])):
        x = rows.double()
        top = x.abs().amax(-1, keepdim=True)
        k = torch.ceil(torch.log2(top.clamp_min(2.0 ** -108) / 448 * (1 - 1e-12)))
        y = x * _two(-k)
        hi = torch.searchsorted(grid, y.abs().contiguous()).clamp(1, 126)
        lo = hi - 1
        up, down = grid[hi] - y.abs(), y.abs() - grid[lo]
        pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
        stored = torch.sign(y) * grid[pick] * _two(k)
        every = _value8(data.view(torch.uint8)) * _two(exps.long() - 127).transpose(1, 2).unsqueeze(-1)
        every = every.flatten(0, 1)
        every[s["slots"].long()] = stored
        every = every.view(data.shape)
        parts = [every[table[b, :_ceil(cu[b + 1] - cu[b], block)].long()].flatten(0, 1)[:cu[b + 1] - cu[b]]
                 for b in range(len(cu) - 1)]
        out.append(torch.cat(parts))
    return out


def exact(case, seed):
    if case["op"] == "decode":
        return _exact_decode(prepare(case, seed))
    if case["op"] == "rows":
        return _exact_rows(prepare(case, seed))
    return None  # pages are moved and counted: nothing is rounded
