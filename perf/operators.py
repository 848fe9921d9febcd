"""Operators of beam search over a paged key-value cache, as cases that can be timed and checked.

Kinds:

    attend     attention over a paged cache: one new token (or a few) per sequence, or prompts whose rows are ragged; grouped heads,
               optionally a sliding window and the first tokens that stay visible beside it; with "append" the new rows' keys and values
               are written to the cache first
    beam       selection over beams and vocabulary from a step's logits
    states     recurrent states of several layers reordered to the beams that were kept, in place
    step       a beam step of the cache: sequences take over their parents' pages and get room for a row, for which pages that others
               hold too are copied
    compact    live pages move to the front of the pools

Where ``own`` is false ``run`` computes them by elementary torch operations in 32 bits (in 64 where scores of different beams are compared),
where it is true through the entry points of the C ABI.
"""
import ctypes as C
import math

import numpy as np
import torch

own = False

SINGLE = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one user of a 12-head model in the middle of a conversation: latency only
        {"name": "token_1", "kind": "attend", "sequences": 1, "chunk": 1, "heads": 12, "kv_heads": 12, "dim": 64, "longest": 700, "page_rows": 16,
         "window": 0, "sinks": 0, "ragged": False, "append": False, "dtype": "bf16"},
        # a serving batch with grouped heads, every sequence somewhere else
        {"name": "token_32", "kind": "attend", "sequences": 32, "chunk": 1, "heads": 32, "kv_heads": 8, "dim": 128, "longest": 4096, "page_rows": 16,
         "window": 0, "sinks": 0, "ragged": False, "append": False, "dtype": "bf16"},
        # documents: long caches, the most bytes
        {"name": "token_long", "kind": "attend", "sequences": 16, "chunk": 1, "heads": 32, "kv_heads": 8, "dim": 128, "longest": 32768,
         "page_rows": 64, "window": 0, "sinks": 0, "ragged": False, "append": False, "dtype": "bf16"},
        # endless conversations: a window and the first tokens, three ids per sequence to be verified at once
        {"name": "token_window", "kind": "attend", "sequences": 64, "chunk": 3, "heads": 16, "kv_heads": 4, "dim": 64, "longest": 8192,
         "page_rows": 64, "window": 1024, "sinks": 4, "ragged": False, "append": True, "dtype": "bf16"},
        # a 32-bit model of odd widths, pages whose rows are no power of two
        {"name": "token_f32", "kind": "attend", "sequences": 9, "chunk": 1, "heads": 10, "kv_heads": 2, "dim": 80, "longest": 1500, "page_rows": 24,
         "window": 0, "sinks": 0, "ragged": False, "append": False, "dtype": "f32"},
        # prompts of odd lengths admitted behind what their sequences already hold
        {"name": "prompt_window", "kind": "attend", "sequences": 5, "chunk": 777, "heads": 16, "kv_heads": 4, "dim": 64, "longest": 2048,
         "page_rows": 64, "window": 512, "sinks": 4, "ragged": True, "append": True, "dtype": "bf16"},
        # the second half of a long document: the most operations
        {"name": "prompt_long", "kind": "attend", "sequences": 1, "chunk": 6000, "heads": 32, "kv_heads": 8, "dim": 128, "longest": 12000,
         "page_rows": 64, "window": 4096, "sinks": 16, "ragged": False, "append": False, "dtype": "bf16"},
        # one user, four beams
        {"name": "beam_1", "kind": "beam", "groups": 1, "beams": 4, "vocab": 32000, "keep": 4, "dtype": "f32"},
        # a batch of translations, twice as many candidates as beams, odd vocabulary
        {"name": "beam_48", "kind": "beam", "groups": 48, "beams": 6, "vocab": 50021, "keep": 12, "dtype": "f32"},
        # states of twelve recurrent layers (24 heads of 128 x 64) of eight users with four beams
        {"name": "states_8", "kind": "states", "groups": 8, "beams": 4, "layers": 12, "bytes": 24 * 128 * 64 * 4},
        # sixteen users with four beams, caches of a 12-layer model
        {"name": "step_16", "kind": "step", "groups": 16, "beams": 4, "layers": 12, "kv_heads": 12, "dim": 64, "longest": 600, "page_rows": 16},
        # a pool three quarters empty after a busy hour gives its upper part back
        {"name": "compact_4096", "kind": "compact", "sequences": 48, "layers": 4, "kv_heads": 8, "dim": 128, "longest": 640, "page_rows": 32,
         "pool_pages": 4096},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["token", "token", "token", "prompt", "prompt", "beam", "beam", "states", "step", "compact"])
    if kind in ("token", "prompt"):
        dtype = "f32" if kind == "token" and rng.random() < 0.25 else "bf16"
        per = rng.choice([1, 1, 2, 4, 5, 8])
        kv = rng.choice([1, 2, 3, 4, 8, 12] if per < 4 else [1, 2, 4, 8])
        dim = rng.choice([64, 128]) if kind == "prompt" else rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        case = {"kind": "attend", "heads": per * kv, "kv_heads": kv, "dim": dim, "page_rows": rng.choice([16, 24, 32, 64, 128]),
                "window": rng.choice([0, 0, 1]) and _log(rng, 16, 4096), "sinks": rng.choice([0, rng.randint(1, 64)]), "dtype": dtype,
                "append": rng.random() < 0.4}
        if kind == "token":
            case |= {"sequences": _log(rng, 1, 128), "chunk": rng.choice([1, 1, 1, rng.randint(2, 5)]), "ragged": rng.random() < 0.2}
            rows = (1 << 30) // (case["sequences"] * kv * dim * (4 if dtype == "f32" else 2))
            case["longest"] = _log(rng, 16, min(32768, max(32, rows)))
        else:
            case |= {"sequences": _log(rng, 1, 8), "ragged": rng.random() < 0.7}
            case["chunk"] = _log(rng, 17, 6000 // case["sequences"])
            case["longest"] = case["chunk"] + rng.choice([0, _log(rng, 1, 4000)])
        return case
    if kind == "beam":
        beams = rng.randint(1, 12)
        vocab = _log(rng, 500, 130000)
        return {"kind": "beam", "groups": _log(rng, 1, max(1, min(64, (24 << 20) // (beams * vocab)))), "beams": beams, "vocab": vocab,
                "keep": beams * rng.choice([1, 1, 2]), "dtype": rng.choice(["f32", "f32", "bf16"])}
    if kind == "states":
        return {"kind": "states", "groups": _log(rng, 1, 16), "beams": rng.randint(2, 8), "layers": rng.randint(1, 12), "bytes": 16 * _log(rng, 200, 3000)}
    if kind == "step":
        return {"kind": "step", "groups": _log(rng, 1, 32), "beams": rng.randint(2, 8), "layers": rng.randint(1, 12), "kv_heads": rng.choice([1, 2, 4, 12]),
                "dim": rng.choice([64, 128]), "longest": _log(rng, 20, 1000), "page_rows": rng.choice([16, 24, 32, 64])}
    case = {"kind": "compact", "sequences": _log(rng, 1, 64), "layers": rng.randint(1, 4), "kv_heads": rng.choice([1, 4, 8]), "dim": rng.choice([64, 128]),
            "longest": _log(rng, 20, 640), "page_rows": rng.choice([16, 24, 32])}
    return case | {"pool_pages": case["sequences"] * -(-case["longest"] // case["page_rows"]) * rng.randint(2, 4)}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------------


def _spread(rng, count, low, high):
    """`count` whole numbers from `high` down to `low` in equal steps, in any order."""
    return rng.permutation(np.rint(np.linspace(high, max(1, low), count)).astype(np.int64))


def _pages(rng, lengths, page_rows, pool_pages, ld):
    """A table whose sequences hold pages scattered over the pool; what is behind a sequence's pages names no page."""
    need = -(-lengths // page_rows)
    pages = rng.permutation(pool_pages)[:need.sum()]
    table = np.full((len(lengths), ld), 0xffffffff, np.uint32)
    table[np.arange(ld)[None, :] < need[:, None]] = pages
    return table


def _u32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.uint32).view(np.int32)).cuda()


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    state = {"case": case}
    kind = case["kind"]
    if kind == "attend":
        n, kv, dim, rows = case["sequences"], case["kv_heads"], case["dim"], case["page_rows"]
        t = SINGLE[case["dtype"]]
        fresh = _spread(rng, n, case["chunk"] // 3, case["chunk"]) if case["ragged"] else np.full(n, case["chunk"])
        lengths = np.maximum(_spread(rng, n, case["longest"] // 4, case["longest"]), fresh)
        ld = -(-case["longest"] // rows)
        pool = n * ld + 3
        state["starts"] = _u32(np.concatenate([[0], np.cumsum(fresh)])) if case["ragged"] else None
        state["rows"] = int(fresh.sum())
        state["lengths"], state["table"], state["pool_pages"] = _u32(lengths), _u32(_pages(rng, lengths, rows, pool, ld)), pool
        state["q"] = torch.randn(state["rows"], case["heads"], dim, device="cuda", generator=gen).to(t)
        state["k"], state["v"] = (torch.empty(pool, rows, kv, dim, device="cuda", dtype=t).normal_(generator=gen) for _ in range(2))
        state["out"] = torch.empty(state["rows"], case["heads"], dim, device="cuda", dtype=t)
        if case["append"]:
            state["fresh"] = torch.randn(2, state["rows"], kv, dim, device="cuda", generator=gen).to(t)
    elif kind == "beam":
        n = case["groups"] * case["beams"]
        logits = torch.randn(n, case["vocab"], device="cuda", generator=gen) * 2
        # what a grammar forbids, and a few tokens that a trained model is fairly sure of
        logits[torch.rand(n, case["vocab"], device="cuda", generator=gen) < 0.02] = -math.inf
        likely = torch.randint(0, case["vocab"], (n, 8), device="cuda", generator=gen)
        state["logits"] = logits.scatter_add_(1, likely, 6 + 2 * torch.randn(n, 8, device="cuda", generator=gen)).to(SINGLE[case["dtype"]])
        state["scores"] = -torch.rand(n, device="cuda", generator=gen) * 30
        state["finished"] = torch.rand(n, device="cuda", generator=gen) < 0.1
        state["end"] = int(rng.integers(case["vocab"]))
        shape = (case["groups"], case["keep"])
        state["next"] = [torch.empty(shape, device="cuda", dtype=t) for t in (torch.float32, torch.int32, torch.int32, torch.bool)]
    elif kind == "states":
        n = case["groups"] * case["beams"]
        state["states"] = [torch.randn(n, case["bytes"] // 4, device="cuda", generator=gen) for _ in range(case["layers"])]
        state["parents"] = _u32(_parents(rng, case))
    else:
        n = case["sequences"] if kind == "compact" else case["groups"] * case["beams"]
        rows, width = case["page_rows"], case["kv_heads"] * case["dim"]
        if kind == "compact":
            lengths, pool = _spread(rng, n, case["longest"] // 4, case["longest"]), case["pool_pages"]
        else:
            # the beams of a group stand at the same place, their first pages are the prompt's
            lengths = np.repeat(_spread(rng, case["groups"], case["longest"] // 4, case["longest"]), case["beams"])
            pool = n * (-(-case["longest"] // rows) + 2)
            state["parents"] = _u32(_parents(rng, case))
        ld = case["longest"] // rows + 2
        table = _pages(rng, lengths, rows, pool, ld)
        if kind == "step":
            first = np.arange(n) // case["beams"] * case["beams"]
            shared = np.arange(ld)[None, :] < (lengths // rows // 2)[:, None]
            table = np.where(shared, table[first], table)
        live = table[np.arange(ld)[None, :] < (-(-lengths // rows))[:, None]]
        # table, lengths and how many entries hold a page, in one buffer; `start` is what a pass sets out from
        state["start"] = _u32(np.concatenate([table.reshape(-1), lengths.astype(np.uint32), np.bincount(live, minlength=pool).astype(np.uint32)]))
        state["book"] = state["start"].clone()
        state["pool"] = torch.empty(2 * case["layers"], pool, rows, width, device="cuda", dtype=torch.bfloat16).normal_(generator=gen)
    return state


def _parents(rng, case):
    """Which beam of its group each kept candidate continues: the better ones more often than the others."""
    beams = case["beams"]
    chosen = np.sort((rng.random((case["groups"], beams)) ** 1.5 * beams).astype(np.int64), axis=1)
    return (chosen + np.arange(case["groups"])[:, None] * beams).reshape(-1)


def _book(state, buffer):
    """table, lengths and holders inside one buffer."""
    case = state["case"]
    n = case["sequences"] if case["kind"] == "compact" else case["groups"] * case["beams"]
    pool = state["pool"].shape[1]
    ld = (buffer.numel() - n - pool) // n
    return buffer[:n * ld].view(n, ld), buffer[n * ld:n * ld + n], buffer[n * ld + n:]


# ---- plain forms -------------------------------------------------------------------------------------------------------------------------------


def _attend(state):
    case = state["case"]
    n, chunk, kv, dim, rows = case["sequences"], case["chunk"], case["kv_heads"], case["dim"], case["page_rows"]
    per, window, sinks = case["heads"] // kv, case["window"], case["sinks"]
    lengths = state["lengths"].long()
    starts = state["starts"].long() if case["ragged"] else torch.arange(n + 1, device="cuda") * chunk
    count = starts[1:] - starts[:-1]
    row = torch.arange(chunk, device="cuda")
    source = (starts[:-1, None] + row).clamp(max=state["rows"] - 1)
    if case["append"]:
        sequence = torch.repeat_interleave(torch.arange(n, device="cuda"), count, output_size=state["rows"])
        to = (lengths - starts[1:])[sequence] + torch.arange(state["rows"], device="cuda")
        page = state["table"].long()[sequence, to // rows]
        state["k"][page, to % rows] = state["fresh"][0]
        state["v"][page, to % rows] = state["fresh"][1]
    # keys that some row sees: the first ones, and those from the first row's window on
    keys = case["longest"]
    if window and sinks + window + chunk < keys:
        keys = sinks + window + chunk
        at = torch.arange(keys, device="cuda")
        first = (lengths - count + 1 - window).clamp(min=sinks)
        at = torch.where(at < sinks, at, first[:, None] + at - sinks)
    else:
        at = torch.arange(keys, device="cuda").expand(n, keys)
    real = at < lengths[:, None]
    page = state["table"].long().gather(1, (at // rows).clamp(max=state["table"].shape[1] - 1))
    place = torch.where(real, page * rows + at % rows, 0)
    # [sequence, head of the cache, row of the group, width]
    k = state["k"].view(-1, kv, dim)[place].float().transpose(1, 2)
    v = state["v"].view(-1, kv, dim)[place].float().transpose(1, 2)
    q = state["q"].view(-1, kv, per, dim)[source].float().permute(0, 2, 1, 3, 4).reshape(n, kv, chunk * per, dim)
    stands = (lengths - count)[:, None] + row
    seen = real[:, None, :] & (at[:, None, :] <= stands[:, :, None])
    if window:
        seen &= (at[:, None, :] > stands[:, :, None] - window) | (at[:, None, :] < sinks)
    score = (q @ k.transpose(2, 3) * dim ** -0.5).view(n, kv, chunk, per, keys)
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(n, kv, chunk * per, keys) @ v).view(n, kv, chunk, per, dim) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 2, 1, 3, 4).reshape(n, chunk, kv * per, dim)
    if case["ragged"]:
        out = out[row < count[:, None]]
    out = out.reshape(-1, kv * per, dim).to(state["q"].dtype)
    return (out, state["k"], state["v"]) if case["append"] else out


def _beam(state):
    case = state["case"]
    groups, beams, vocab, keep = case["groups"], case["beams"], case["vocab"], case["keep"]
    # scores of different beams lie next to each other: in 64 bits
    logits = state["logits"].double().view(groups, beams, vocab)
    top = logits.amax(-1, keepdim=True)
    total = top + (logits - top).exp().sum(-1, keepdim=True).log()
    scores, finished = state["scores"].double().view(groups, beams, 1), state["finished"].view(groups, beams, 1)
    alive = ~finished & torch.isfinite(total)
    score = torch.where(alive, scores + (logits - total), -math.inf)
    end = torch.arange(vocab, device="cuda") == state["end"]
    score = torch.where(finished & end, scores, score).view(groups, beams * vocab)
    best, at = score.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :keep], at[:, :keep]
    beam, token = at // vocab, at % vocab
    parents = beam + torch.arange(groups, device="cuda")[:, None] * beams
    done = state["finished"][parents] | (token == state["end"])
    return best.float(), token.int(), parents.int(), done


def _states(state):
    parents = state["parents"].long()
    return [s.copy_(s[parents]) for s in state["states"]]


def _step(state):
    case = state["case"]
    rows, n = case["page_rows"], case["groups"] * case["beams"]
    table, lengths, holders = (t.long() for t in _book(state, state["start"]))
    pool, ld = state["pool"], table.shape[1]
    parents = state["parents"].long()
    column = torch.arange(ld, device="cuda")
    # the parents' pages and lengths; entries behind the last page stay what they were
    lengths = lengths[parents]
    live = column < -(-lengths // rows)[:, None]
    table = torch.where(live, table[parents], table)
    holders = torch.bincount(table[live], minlength=holders.numel())
    # one row more: a page of its own where the last one is full, a copy where others hold it and an earlier one of them keeps it
    last = table.gather(1, ((lengths - 1) // rows)[:, None])[:, 0]
    order = torch.arange(n, device="cuda")
    keeper = torch.full_like(holders, n).scatter_reduce(0, last, order, "amin")
    opens = lengths % rows == 0
    copies = ~opens & (holders[last] > 1) & (keeper[last] != order)
    needs = opens | copies
    free = torch.cat([torch.nonzero(holders == 0)[:, 0], torch.zeros(n, dtype=torch.long, device="cuda")])
    page = torch.where(needs, free[(needs.cumsum(0) - 1).clamp(min=0)], last)
    pool[:, page[copies]] = pool[:, last[copies]]
    holders = holders.scatter_add(0, last, -copies.long()).scatter_add(0, page, needs.long())
    table = table.scatter(1, (lengths // rows)[:, None], page[:, None])
    state["book"].copy_(torch.cat([table.reshape(-1), lengths + 1, holders]))
    return state["book"], pool


def _compact(state):
    rows = state["case"]["page_rows"]
    table, lengths, holders = (t.long() for t in _book(state, state["start"]))
    live = holders > 0
    count = live.sum()
    index = torch.arange(holders.numel(), device="cuda")
    low = torch.nonzero(~live & (index < count))[:, 0]
    high = torch.nonzero(live & (index >= count))[:, 0]
    state["pool"][:, low] = state["pool"][:, high]
    moved = index.scatter(0, high, low)
    holders = holders.scatter(0, low, holders[high]).scatter(0, high, 0)
    held = torch.arange(table.shape[1], device="cuda") < -(-lengths // rows)[:, None]
    table = torch.where(held, moved[table.clamp(0, holders.numel() - 1)], table)
    state["book"].copy_(torch.cat([table.reshape(-1), lengths, holders]))
    return state["book"], state["pool"], count.int()


# ---- the framework's operators -----------------------------------------------------------------------------------------------------------------


def _bind(state):
    """The calls of a pass, as a program that keeps its buffers makes them step after step."""
    from tnsr_b200 import _native
    lib, case, kind = _native.lib(), state["case"], state["case"]["kind"]

    def at(t):
        return None if t is None else t.data_ptr()

    def scratch(nbytes):
        return torch.zeros(max(int(nbytes), 1), dtype=torch.uint8, device="cuda")

    def call(entry, *args):
        return lambda stream: _native.check(entry(*args, stream))

    keep = state["kept"] = []
    dtype = _native.DTYPE[case.get("dtype", "bf16")]
    if kind == "attend":
        dim = case["dim"]
        work = scratch(lib.tnsr_b200_paged_attention_workspace(dim, dim, dtype))
        args = _native.PagedAttentionArgs(
            q=at(state["q"]), k_pool=at(state["k"]), v_pool=at(state["v"]), table=at(state["table"]), lengths=at(state["lengths"]),
            row_starts=at(state["starts"]), out=at(state["out"]), workspace=at(work), workspace_bytes=work.numel(), sequences=case["sequences"],
            chunk=case["chunk"], rows=state["rows"], q_ld=case["heads"] * dim, out_ld=case["heads"] * dim, heads=case["heads"],
            kv_heads=case["kv_heads"], dim=dim, vdim=dim, table_ld=state["table"].shape[1], page_rows=case["page_rows"],
            pool_pages=state["pool_pages"], window=case["window"], sinks=case["sinks"] if case["window"] else 0, scale=dim ** -0.5, dtype=dtype)
        keep += [work, args]
        calls = [call(lib.tnsr_b200_paged_attention, C.byref(args))]
        if not case["append"]:
            return calls, state["out"]
        fresh = _native.PagedAppendArgs(
            k=at(state["fresh"][0]), v=at(state["fresh"][1]), k_pool=at(state["k"]), v_pool=at(state["v"]), table=at(state["table"]),
            lengths=at(state["lengths"]), row_starts=at(state["starts"]), sequences=case["sequences"], chunk=case["chunk"], rows=state["rows"],
            k_ld=case["kv_heads"] * dim, v_ld=case["kv_heads"] * dim, kv_heads=case["kv_heads"], dim=dim, vdim=dim, table_ld=state["table"].shape[1],
            page_rows=case["page_rows"], pool_pages=state["pool_pages"], dtype=dtype)
        keep.append(fresh)
        return [call(lib.tnsr_b200_paged_append, C.byref(fresh))] + calls, (state["out"], state["k"], state["v"])
    if kind == "beam":
        scores, tokens, parents, done = state["next"]
        work = scratch(lib.tnsr_b200_beam_select_workspace(case["groups"], case["beams"], case["vocab"], case["keep"]))
        args = _native.BeamSelectArgs(
            logits=at(state["logits"]), scores=at(state["scores"]), finished=at(state["finished"]), next_scores=at(scores), tokens=at(tokens),
            parents=at(parents), next_finished=at(done), workspace=at(work), workspace_bytes=work.numel(), logits_ld=case["vocab"],
            groups=case["groups"], beams=case["beams"], vocab=case["vocab"], keep=case["keep"], end_token=state["end"], dtype=dtype)
        keep += [work, args]
        return [call(lib.tnsr_b200_beam_select, C.byref(args))], tuple(state["next"])
    if kind == "states":
        count = case["layers"]
        tensors = (C.c_void_p * count)(*[at(t) for t in state["states"]])
        nbytes = (C.c_uint64 * count)(*[case["bytes"]] * count)
        keep += [tensors, nbytes]
        return [call(lib.tnsr_b200_reorder_states, tensors, nbytes, nbytes, count, at(state["parents"]), case["groups"], case["beams"], None)], state["states"]
    table, lengths, holders = _book(state, state["book"])
    count, pool_pages = 2 * case["layers"], state["pool"].shape[1]
    tensors = (C.c_void_p * count)(*[at(state["pool"][i]) for i in range(count)])
    nbytes = (C.c_uint64 * count)(*[state["pool"][0, 0].numel() * 2] * count)
    work = scratch(lib.tnsr_b200_pages_workspace(table.shape[0], pool_pages))
    book = _native.PageBook(table=at(table), lengths=at(lengths), holders=at(holders), workspace=at(work), workspace_bytes=work.numel(),
                            sequences=table.shape[0], table_ld=table.shape[1], page_rows=case["page_rows"], pool_pages=pool_pages)
    pools = _native.PagePools(tensors=tensors, page_bytes=nbytes, count=count)
    keep += [tensors, nbytes, work, book, pools]
    if kind == "compact":
        live = torch.empty((), dtype=torch.int32, device="cuda")
        return [call(lib.tnsr_b200_pages_compact, C.byref(book), C.byref(pools), at(live))], (state["book"], state["pool"], live)
    calls = [call(lib.tnsr_b200_pages_fork, C.byref(book), at(state["parents"])),
             call(lib.tnsr_b200_pages_reserve, C.byref(book), C.byref(pools), None, 1)]
    return calls, (state["book"], state["pool"])


def run(state):
    if own:
        if "bound" not in state:
            state["bound"] = _bind(state)
        if "start" in state:      # every pass sets out from the same place
            state["book"].copy_(state["start"])
        calls, outputs = state["bound"]
        stream = torch.cuda.current_stream().cuda_stream
        for c in calls:
            c(stream)
        return outputs
    return {"attend": _attend, "beam": _beam, "states": _states, "step": _step, "compact": _compact}[state["case"]["kind"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "attend":
        n, width = case["sequences"], 4 if case["dtype"] == "f32" else 2
        # rows and lengths as prepare() spreads them, on average beside the longest
        chunk = (max(1, case["chunk"] // 3) + case["chunk"]) / 2 if case["ragged"] else case["chunk"]
        rest = max(chunk, (max(1, case["longest"] // 4) + case["longest"]) / 2)
        nbytes = flops = 0.0
        for length, many in ((case["longest"], 1), (rest, n - 1)):
            keys, pairs = length, chunk * (length - (chunk - 1) / 2)
            if case["window"]:
                seen = case["sinks"] + case["window"]
                keys = min(length, seen + chunk - 1)
                start = length - chunk + 1      # keys before the first row's end
                full = min(chunk, max(0.0, length - seen))      # rows that see the window and the first tokens and no more
                pairs = full * seen + (chunk - full) * (start + min(seen, length)) / 2 if full < chunk else chunk * seen
            if case["append"]:
                nbytes += many * chunk * case["kv_heads"] * case["dim"] * 2 * width
            nbytes += many * keys * case["kv_heads"] * case["dim"] * 2 * width + many * chunk * case["heads"] * case["dim"] * 2 * width
            flops += many * pairs * case["heads"] * case["dim"] * 4
        return {"bytes": nbytes, "flops": flops}
    if kind == "beam":
        elements = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": elements * (4 if case["dtype"] == "f32" else 2) + case["groups"] * case["keep"] * 13, "flops": elements * 4}
    beams = case.get("beams", 1)
    if kind in ("states", "step"):
        # how often beam j is a parent: its share of the interval under the power that _parents() raises to
        share = [((j + 1) / beams) ** (2 / 3) - (j / beams) ** (2 / 3) for j in range(beams)]
        distinct = sum(1 - (1 - s) ** beams for s in share)
    if kind == "states":
        # rows whose parent is another one are written, what they come from is read once
        return {"bytes": case["groups"] * case["layers"] * case["bytes"] * (2 * max(1.0, distinct - 1)), "flops": 0}
    width = case["kv_heads"] * case["dim"] * 2
    page = 2 * case["layers"] * case["page_rows"] * width
    if kind == "step":
        n, entries = case["groups"] * beams, 0.625 * case["longest"] / case["page_rows"]
        copies = case["groups"] * (beams - distinct) * (1 - 1 / case["page_rows"])
        return {"bytes": n * entries * 8 + copies * 2 * page, "flops": 0}
    need = case["sequences"] * 0.625 * case["longest"] / case["page_rows"]
    return {"bytes": 2 * need * (1 - need / case["pool_pages"]) * page + 8 * need + 8 * case["pool_pages"], "flops": 0}


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "attend":
        lengths, table = state["lengths"].tolist(), state["table"]
        starts = state["starts"].tolist() if case["ragged"] else [i * case["chunk"] for i in range(case["sequences"] + 1)]
        out = torch.zeros(state["rows"], case["heads"], case["dim"], dtype=torch.float64, device="cuda")
        per = case["heads"] // case["kv_heads"]
        for s, length in enumerate(lengths):
            for i in range(starts[s], starts[s + 1]) if case["append"] else ():
                j = length - starts[s + 1] + i
                for n, fresh in zip("kv", state["fresh"]):
                    state[n][table[s, j // case["page_rows"]], j % case["page_rows"]] = fresh[i]
            if not length or starts[s + 1] == starts[s]:
                continue
            pages = table[s, :-(-length // case["page_rows"])].long()
            place = torch.arange(length - (starts[s + 1] - starts[s]), length, device="cuda")[:, None]
            j = torch.arange(length, device="cuda")[None, :]
            hidden = j > place
            if case["window"]:
                hidden |= (j + case["window"] <= place) & (j >= case["sinks"])
            for h in range(case["heads"]):
                k, v = (state[n][pages, :, h // per].reshape(-1, case["dim"])[:length].double() for n in "kv")
                logits = torch.einsum("id,jd->ij", state["q"][starts[s]:starts[s + 1], h].double(), k) / math.sqrt(case["dim"])
                weights = torch.softmax(logits.masked_fill(hidden, -math.inf), dim=1)
                out[starts[s]:starts[s + 1], h] = torch.nan_to_num(weights, nan=0.0) @ v
        return (out, state["k"], state["v"]) if case["append"] else out
    if kind == "beam":
        keep, vocab, beams = case["keep"], case["vocab"], case["beams"]
        scores, finished = state["scores"].double(), state["finished"].tolist()
        best = torch.empty(case["groups"], keep, dtype=torch.float64, device="cuda")
        for g in range(case["groups"]):
            rows = []
            for b in range(g * beams, (g + 1) * beams):
                row = scores[b] + torch.log_softmax(state["logits"][b].double(), 0)
                if finished[b]:
                    row = torch.full_like(row, -math.inf)
                    row[state["end"]] = scores[b]
                rows.append(row)
            best[g] = torch.topk(torch.cat(rows), keep).values
        return best, None, None, None
    if kind == "states":
        parents = state["parents"].tolist()
        return [torch.stack([s[p] for p in parents]).double() for s in state["states"]]
    rows = case["page_rows"]
    table, lengths, holders = (t.cpu().numpy().view(np.uint32).astype(np.int64).copy() for t in _book(state, state["start"]))
    pool = state["pool"]
    if kind == "compact":
        count = int((holders > 0).sum())
        free = [p for p in range(count) if holders[p] == 0]
        for low, high in zip(free, [p for p in range(count, len(holders)) if holders[p]]):
            pool[:, low] = pool[:, high]
        return None, pool, None
    parents = state["parents"].tolist()
    table, lengths = [list(table[p]) for p in parents], [int(lengths[p]) for p in parents]
    held = {}
    for s, length in enumerate(lengths):
        for p in table[s][:-(-length // rows)]:
            held.setdefault(p, []).append(s)
    free = (p for p in range(len(holders)) if p not in held)
    for s, length in enumerate(lengths):
        slot = length // rows
        if length % rows == 0:
            table[s][slot] = next(free)
        elif held[table[s][slot]][0] != s:
            page = next(free)
            pool[:, page] = pool[:, table[s][slot]]
            table[s][slot] = page
    return None, pool
