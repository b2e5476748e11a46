"""A serving step over a paged 8-bit key/value cache, as measurable cases.

Four operators that are used one after another, beside the framework's attention over plain rows:

* ``gatgpu_rotate_forward`` / ``_backward``: the RMS norm of each head's query and key and the rotation by its
  position in one pass, with the gradients of the rows and of the norms' weights.
* ``gatgpu_blocks_assign``: block tables, slots, positions, row offsets and lengths of a step, from the requests'
  lengths on the GPU, with pages taken from a free list, to which ``gatgpu_blocks_release`` gives those of requests
  that ended.
* ``gatgpu_cache_append``: keys and values into their pages as e4m3 bytes, with a power of two as the scale of each
  page and head.
* ``gatgpu_cache_attention``: causal attention of each request's new rows over its pages.

A page holds ``page`` tokens: keys as [kv head][token][dim], values as [kv head][dim][token].  Lengths of a case come
from the case alone (``lengths`` seeds them), so that its work does not depend on the inputs' seed.
"""
import math
import os
import random
import sys

import torch

own = False

if os.path.join(os.getcwd(), "gat-tfs_amd") not in sys.path:
    sys.path.insert(0, os.path.join(os.getcwd(), "gat-tfs_amd"))

DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}
TOP = 448.0  # largest e4m3 value
LEAST, MOST = -64, 64  # exponents of scales


def _rotate(name, rows, heads, kv_heads, dim, rot, precision, train, pairs="halves", far=4096):
    """far: positions are below it; rot: how many of a head's columns turn."""
    return {"name": name, "kind": "rotate", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "precision": precision, "train": train, "pairs": pairs, "far": far}


def _blocks(name, requests, page, cached, fresh, ended, lengths):
    """cached, fresh: most tokens in the cache and to come; fresh 1: one each; ended: requests that ended before the step."""
    return {"name": name, "kind": "blocks", "requests": requests, "page": page, "cached": cached, "fresh": fresh,
            "ended": ended, "lengths": lengths}


def _append(name, requests, page, kv_heads, dim, fresh, precision, lengths):
    return {"name": name, "kind": "append", "requests": requests, "page": page, "kv_heads": kv_heads, "dim": dim,
            "fresh": fresh, "precision": precision, "lengths": lengths}


def _attend(name, requests, lo, hi, rows_lo, rows_hi, heads, kv_heads, dim, page, precision, lengths):
    return {"name": name, "kind": "attend", "requests": requests, "lo": lo, "hi": hi, "rows_lo": rows_lo,
            "rows_hi": rows_hi, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "precision": precision,
            "lengths": lengths}


def listed():
    return [
        # The rows of a few new tokens at far positions: the smallest call of a serving loop.
        _rotate("rotate_tokens_7", 7, 8, 8, 64, 64, "bf16", False, far=200_000),
        # A packed training batch in front of the attention over its segments.
        _rotate("rotate_train_20k", 20_011, 16, 4, 128, 128, "bf16", True),
        # Narrow heads in FP32, half of each turned, neighbouring columns as pairs.
        _rotate("rotate_train_fp32_6k", 6_007, 8, 8, 32, 16, "fp32", True, pairs="neighbours"),
        # One decoding step of a small batch.
        _blocks("blocks_step_12", 12, 16, 3_000, 1, 0, 1),
        # Prompts of many requests at once, after hundreds of others have ended.
        _blocks("blocks_prompts_2500", 2_500, 16, 900, 1_200, 300, 2),
        # The new token of each request, into pages of which most are partly full.
        _append("append_step_96", 96, 32, 8, 128, 1, "bf16", 3),
        # Prompts of two dozen requests.
        _append("append_prompts_24", 24, 64, 8, 128, 6_000, "bf16", 4),
        # One new token of one request over a short cache.
        _attend("cached_token_900", 1, 900, 900, 1, 1, 8, 8, 64, 16, "bf16", 5),
        # One new token of one request over a very long cache.
        _attend("cached_token_260k", 1, 260_001, 260_001, 1, 1, 32, 8, 128, 64, "bf16", 6),
        # One new token of each of 48 requests of very different lengths, key/value heads shared by four.
        _attend("cached_tokens_48x24k", 48, 200, 24_000, 1, 1, 32, 8, 128, 32, "bf16", 7),
        # A few drafted tokens of each request are looked at in one pass, in FP32.
        _attend("cached_drafts_fp32", 20, 90, 6_000, 2, 5, 8, 2, 64, 16, "fp32", 8),
        # Chunks of prompts over what their requests hold already: the largest call.
        _attend("cached_chunks_6x2k", 6, 1_500, 14_000, 300, 2_000, 16, 4, 128, 64, "bf16", 9),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    precision = rng.choice(("bf16", "bf16", "bf16", "fp32"))
    kv_heads, group = rng.choice(((8, 1), (8, 4), (4, 4), (2, 4), (1, 8), (3, 2), (2, 7), (5, 1)))
    dim = rng.choice((16, 32, 48, 64, 64, 96, 128, 128))
    page = rng.choice((16, 16, 32, 64, 128))
    kind = rng.choice(("rotate", "blocks", "append", "attend", "attend", "attend"))
    lengths = rng.randrange(1 << 20)
    if kind == "rotate":
        width = (kv_heads * group + kv_heads) * dim
        rows = _log_int(rng, 1, min(60_000, 50_000_000 // width))
        rot = rng.choice((dim, dim, dim // 2))
        return _pure(_rotate("", rows, kv_heads * group, kv_heads, dim, rot, precision, rng.random() < 0.6,
                             rng.choice(("halves", "halves", "neighbours")), _log_int(rng, 100, 1_000_000)))
    if kind == "blocks":
        requests = _log_int(rng, 1, 3_000)
        fresh = rng.choice((1, 1, _log_int(rng, 4, min(4_000, 2_000_000 // requests))))
        return _pure(_blocks("", requests, page, _log_int(rng, 1, 3_000), fresh, rng.choice((0, 0, 1, 1 + requests // 9)), lengths))
    if kind == "append":
        requests = _log_int(rng, 1, 400)
        fresh = rng.choice((1, 1, _log_int(rng, 2, 8_000_000 // (requests * kv_heads * dim) + 4)))
        return _pure(_append("", requests, page, kv_heads, dim, fresh, precision, lengths))
    hi = _log_int(rng, 20, 60_000)
    requests = _log_int(rng, 1, max(2, min(96, 400_000 // hi)))
    rows = rng.choice((1, 1, 1, 3, 8, _log_int(rng, 16, 1_500)))
    pairs = 1_500_000_000 if precision == "bf16" else 300_000_000
    rows = max(1, min(rows, pairs // (requests * hi * kv_heads * group)))
    return _pure(_attend("", requests, max(1, hi // rng.choice((1, 2, 20))), hi, max(1, rows // rng.choice((1, 3))), rows,
                         kv_heads * group, kv_heads, dim, page, precision, lengths))


def _pure(case):
    return {k: v for k, v in case.items() if k != "name"}


def _lengths(case):
    """Per request: tokens in the cache before the step, and tokens to come; and tokens of the requests that ended."""
    rng = random.Random(case["lengths"])
    n = case["requests"]
    if case["kind"] == "attend":
        total = [_log_int(rng, case["lo"], case["hi"]) for _ in range(n)]
        fresh = [min(_log_int(rng, case["rows_lo"], case["rows_hi"]), t) for t in total]
        return [t - f for t, f in zip(total, fresh)], fresh, []
    if case["kind"] == "append":
        page = case["page"]
        if case["fresh"] == 1:  # open pages, a few of them fresh
            return [rng.randrange(page) for _ in range(n)], [1] * n, []
        return ([rng.choice((0, 0, rng.randrange(page))) for _ in range(n)],
                [_log_int(rng, max(1, case["fresh"] // 8), case["fresh"]) for _ in range(n)], [])
    cached = [rng.choice((0, _log_int(rng, 1, case["cached"]))) for _ in range(n)]
    fresh = [1 if case["fresh"] == 1 else _log_int(rng, 1, case["fresh"]) for _ in range(n)]
    return cached, fresh, [_log_int(rng, 1, case["cached"]) for _ in range(case["ended"])]


def _pages(tokens, page):
    return (tokens + page - 1) // page


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def _exponents(amax):
    """The least e with amax <= 448 2^e, within the scales' range."""
    m, x = torch.frexp(amax)  # amax = m 2^x, m in [1/2, 1); 448 = 7/8 2^9
    return torch.where(amax > 0, x - 9 + (m > 0.875).int(), LEAST).clamp(LEAST, MOST)


def _table(pages, held, width):
    """A table of `held` of the pages for each request, in their order, -1 behind them."""
    column = torch.arange(width, device="cuda")
    first = torch.tensor([0] + held[:-1]).cumsum(0).cuda()
    index = (first.unsqueeze(1) + column).clamp_max(pages.numel() - 1)
    return torch.where(column < torch.tensor(held, device="cuda").unsqueeze(1), pages[index], -1).contiguous()


def _power(e):
    """2^e, exactly (a library's power function need not be)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _order(pages, g):
    return torch.randperm(pages, generator=g, device="cuda").to(torch.int32)


def _rotate_state(case, g):
    t = DTYPE[case["precision"]]
    rows, h, hk, d, rot = case["rows"], case["heads"], case["kv_heads"], case["dim"], case["rot"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    qkv = normal(rows, h + 2 * hk, d).to(t)  # one projection's rows: the values pass by
    state = {"q": qkv[:, :h], "k": qkv[:, h:h + hk], "gamma_q": 1 + 0.2 * normal(d), "gamma_k": 1 + 0.2 * normal(d),
             "eps": 1e-6, "position": torch.randint(0, case["far"], (rows,), generator=g, device="cuda", dtype=torch.int32),
             "freq": torch.pow(10000.0, -2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot).cuda()}
    if case["train"]:
        dy = normal(rows, h + hk, d).to(t)
        state["dq"], state["dk"] = dy[:, :h], dy[:, h:]
    return state


def _blocks_state(case, g):
    before, fresh, ended = _lengths(case)
    page = case["page"]
    held, gone = [_pages(b, page) for b in before], [_pages(e, page) for e in ended]
    total = [_pages(b + f, page) for b, f in zip(before, fresh)]
    taken, rows = sum(total) - sum(held), sum(fresh)
    spare = max(1, taken - sum(gone) // 2)  # free before the call: with the ended requests' pages, enough
    order = _order(sum(held) + sum(gone) + spare, g)
    pages = order.numel()
    free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    free[:spare] = order[sum(held) + sum(gone):]
    state = {"page": page, "pages": pages, "rows": rows + rows // 8 + 1, "cached": _ints(before), "fresh": _ints(fresh),
             "table": _table(order, held, max(total)), "free": free, "free_count": _ints([spare])}
    if ended:
        state["ended"] = _ints(ended)
        state["ended_table"] = _table(order[sum(held):], gone, max(gone))
    return state


def _append_state(case, g):
    t = DTYPE[case["precision"]]
    before, fresh, _ = _lengths(case)
    page, hk, d = case["page"], case["kv_heads"], case["dim"]
    held = [_pages(b + f, page) for b, f in zip(before, fresh)]
    pages = sum(held)
    table = _table(_order(pages, g), held, max(held))
    rows = sum(fresh)
    q_begin = _offsets(fresh)
    at = torch.arange(rows, device="cuda")
    request = torch.searchsorted(q_begin[1:].contiguous(), at, right=True)
    pos = at - q_begin[request] + _ints(before)[request]
    slot = (table[request, pos // page] * page + pos % page).to(torch.int32)
    kv = torch.randn(rows, 2 * hk, d, generator=g, device="cuda")
    kv[:, :, :: max(1, d // 4)] *= 4  # a few columns are larger than the others, as keys' are
    kv = kv.to(t)
    k = torch.randint(0, 127, (pages, hk, page, d), generator=g, device="cuda", dtype=torch.uint8)
    v = torch.randint(0, 127, (pages, hk, d, page), generator=g, device="cuda", dtype=torch.uint8)
    scales = [_power(torch.randint(-9, -5, (pages, hk), generator=g, device="cuda")) for _ in range(2)]
    return {"k_new": kv[:, :hk], "v_new": kv[:, hk:], "slot": slot, "k": k, "v": v, "k_scale": scales[0],
            "v_scale": scales[1], "page": page, "pages": pages}


def _quantized(x, dims):
    """Bytes and scales of whole pages: one scale for what `dims` span."""
    e = _exponents(x.abs().amax(dims, keepdim=True))
    return (x * _power(-e)).to(torch.float8_e4m3fn).view(torch.uint8), _power(e[:, :, 0, 0])


def _attend_state(case, g):
    t = DTYPE[case["precision"]]
    before, fresh, _ = _lengths(case)
    page, h, hk, d = case["page"], case["heads"], case["kv_heads"], case["dim"]
    held = [_pages(b + f, page) for b, f in zip(before, fresh)]
    pages, width = sum(held), max(held)
    state = {"page": page, "pages": pages, "table": _table(_order(pages, g), held, width), "width": width, "q_begin": _offsets(fresh),
             "k_len": _ints([b + f for b, f in zip(before, fresh)]), "most": max(fresh)}
    state["q"] = torch.randn(sum(fresh), h, d, generator=g, device="cuda").to(t)
    state["k"], state["k_scale"] = _quantized(torch.randn(pages, hk, page, d, generator=g, device="cuda"), (2, 3))
    state["v"], state["v_scale"] = _quantized(torch.randn(pages, hk, d, page, generator=g, device="cuda"), (2, 3))
    return state


_STATES = {"rotate": _rotate_state, "blocks": _blocks_state, "append": _append_state, "attend": _attend_state}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = _STATES[case["kind"]](case, g)
    state["case"] = case
    if own:
        _keep(state)
    return state


_context = None


def _cache(state):
    import gatgpu

    case = state["case"]
    return gatgpu.Cache(pages=state["pages"], page=state["page"], kv_heads=case["kv_heads"], dim=case["dim"],
                        k=state["k"].data_ptr(), v=state["v"].data_ptr(), k_scale=state["k_scale"].data_ptr(),
                        v_scale=state["v_scale"].data_ptr())


def _keep(state):
    """The output buffers, workspace and call descriptions that a program keeps."""
    global _context
    import gatgpu

    if _context is None:
        _context = gatgpu.Context(0)
    case = state["case"]
    precision = gatgpu.BF16 if case.get("precision") == "bf16" else gatgpu.FP32
    need = 0
    if case["kind"] == "rotate":
        q, k = state["q"], state["k"]
        h = case["heads"]
        y = torch.empty(q.shape[0], h + case["kv_heads"], case["dim"], dtype=q.dtype, device="cuda")
        out = {"q": y[:, :h], "k": y[:, h:]}
        io = gatgpu.RotateIO(precision=precision, heads=h, kv_heads=case["kv_heads"], dim=case["dim"], norm=1,
                             rot=case["rot"], pairs=gatgpu.PAIRS_HALVES if case["pairs"] == "halves" else gatgpu.PAIRS_NEIGHBOURS,
                             eps=state["eps"], rows=q.shape[0], q=q.data_ptr(), q_stride=q.stride(0), k=k.data_ptr(),
                             k_stride=k.stride(0), gamma_q=state["gamma_q"].data_ptr(), gamma_k=state["gamma_k"].data_ptr(),
                             position=state["position"].data_ptr(), freq=state["freq"].data_ptr(),
                             q_out=out["q"].data_ptr(), q_out_stride=y.stride(0), k_out=out["k"].data_ptr(),
                             k_out_stride=y.stride(0))
        if case["train"]:
            dx = torch.empty_like(y)
            out["dq"], out["dk"] = dx[:, :h], dx[:, h:]
            out["dgamma_q"], out["dgamma_k"] = torch.empty_like(state["gamma_q"]), torch.empty_like(state["gamma_k"])
            io.dq_out, io.dk_out = state["dq"].data_ptr(), state["dk"].data_ptr()
            io.dq_out_stride, io.dk_out_stride = state["dq"].stride(0), state["dk"].stride(0)
            io.dq, io.dk, io.dq_stride, io.dk_stride = out["dq"].data_ptr(), out["dk"].data_ptr(), dx.stride(0), dx.stride(0)
            io.dgamma_q, io.dgamma_k = out["dgamma_q"].data_ptr(), out["dgamma_k"].data_ptr()
            need = _context.rotate_workspace(io)
    elif case["kind"] == "blocks":
        n, rows = case["requests"], state["rows"]
        out = {"table": state["table"], "free": state["free"]}
        for name, size in (("free_left", 1), ("stored", n), ("k_len", n), ("q_begin", n + 1), ("slot", rows), ("position", rows), ("unserved", 1)):
            out[name] = torch.empty(size, dtype=torch.int32, device="cuda")
        count = state["free_count"]
        if case["ended"]:
            table, count = state["ended_table"], torch.empty_like(count)
            state["given"] = count
            state["release"] = gatgpu.BlocksIO(requests=case["ended"], page=state["page"], pages=state["pages"], blocks=table.shape[1],
                                               table_stride=table.stride(0), cached=state["ended"].data_ptr(), table=table.data_ptr(),
                                               free=state["free"].data_ptr(), free_count=state["free_count"].data_ptr(),
                                               free_left=count.data_ptr())
            need = _context.blocks_workspace(state["release"])
        io = gatgpu.BlocksIO(requests=n, page=state["page"], pages=state["pages"], rows=rows, blocks=state["table"].shape[1],
                             table_stride=state["table"].stride(0), cached=state["cached"].data_ptr(), fresh=state["fresh"].data_ptr(),
                             free_count=count.data_ptr(), **{name: t.data_ptr() for name, t in out.items()})
        need = max(need, _context.blocks_workspace(io))
    elif case["kind"] == "append":
        k, v = state["k_new"], state["v_new"]
        out = {"k": state["k"].view(torch.float8_e4m3fn), "v": state["v"].view(torch.float8_e4m3fn),
               "k_scale": state["k_scale"], "v_scale": state["v_scale"]}
        io = gatgpu.AppendIO(precision=precision, rows=k.shape[0], k=k.data_ptr(), k_stride=k.stride(0), v=v.data_ptr(),
                             v_stride=v.stride(0), slot=state["slot"].data_ptr())
    else:
        q = state["q"]
        out = {"out": torch.empty_like(q), "lse": torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")}
        io = gatgpu.CacheAttentionIO(precision=precision, heads=case["heads"], scale=1 / math.sqrt(case["dim"]), rows=q.shape[0],
                                     requests=case["requests"], most=state["most"], blocks=state["width"],
                                     table_stride=state["table"].stride(0), q=q.data_ptr(), q_stride=q.stride(0),
                                     q_begin=state["q_begin"].data_ptr(), k_len=state["k_len"].data_ptr(),
                                     table=state["table"].data_ptr(), out=out["out"].data_ptr(), out_stride=out["out"].stride(0),
                                     lse=out["lse"].data_ptr())
        need = _context.cache_attention_workspace(_cache(state), io)
    state["work"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    state.update(io=io, outputs=out)


def run(state):
    kind = state["case"]["kind"]
    if own:
        io, work = state["io"], state["work"]
        if kind == "rotate":
            _context.rotate_forward(io)
            if state["case"]["train"]:
                _context.rotate_backward(io, work.data_ptr(), work.numel())
        elif kind == "blocks":
            if "release" in state:
                _context.blocks_release(state["release"], work.data_ptr(), work.numel())
            _context.blocks_assign(io, work.data_ptr(), work.numel())
        elif kind == "append":
            _context.cache_append(_cache(state), io)
        else:
            _context.cache_attention(_cache(state), io, work.data_ptr(), work.numel())
        return state["outputs"]
    return {"rotate": _plain_rotate, "blocks": _plain_blocks, "append": _plain_append, "attend": _plain_attend}[kind](state)


def _turned(x, cos, sin, rot, pairs):
    """x [rows][heads][dim] with the pairs of its first `rot` columns turned."""
    if pairs == "halves":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_head(x, gamma, eps, cos, sin, case, dy):
    x = x.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * r
    t = DTYPE[case["precision"]]
    y = _turned(n * gamma, cos, sin, case["rot"], case["pairs"]).to(t)
    if dy is None:
        return y, None, None
    dt = _turned(dy.float(), cos, -sin, case["rot"], case["pairs"])
    dgamma = (dt * n).sum((0, 1), dtype=torch.float64).float()
    dn = dt * gamma
    return y, (r * (dn - n * (dn * n).mean(-1, keepdim=True))).to(t), dgamma


def _plain_rotate(state):
    case = state["case"]
    angle = state["position"].double().view(-1, 1, 1) * state["freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out = {}
    out["q"], dq, dgamma_q = _plain_head(state["q"], state["gamma_q"], state["eps"], cos, sin, case, state.get("dq"))
    out["k"], dk, dgamma_k = _plain_head(state["k"], state["gamma_k"], state["eps"], cos, sin, case, state.get("dk"))
    if case["train"]:
        out.update(dq=dq, dk=dk, dgamma_q=dgamma_q, dgamma_k=dgamma_k)
    return out


def _plain_blocks(state):
    page, rows = state["page"], state["rows"]
    table, free, count = state["table"], state["free"], state["free_count"].long()
    requests, width = table.shape
    pages = free.numel()
    if "ended" in state:  # their pages go behind the free ones, in order
        ended = state["ended_table"]
        held = (state["ended"].long() + page - 1) // page
        back = ((torch.arange(ended.shape[1], device="cuda") < held.unsqueeze(1)) & (ended >= 0) & (ended < pages)).flatten()
        place = count + back.cumsum(0) - 1
        room = torch.cat((free, free.new_empty(1)))
        room[torch.where(back & (place < pages), place, pages)] = ended.flatten()
        free = room[:-1]
        count = (count + back.sum()).clamp_max(pages)
    cached, fresh = state["cached"].long(), state["fresh"].long()
    # Pages to take, from the end of the list.
    fits = cached + fresh <= width * page
    had = (cached + page - 1) // page
    need = torch.where(fits, (cached + fresh + page - 1) // page - had, 0)
    upto = need.cumsum(0)
    q_end = fresh.cumsum(0)
    served = fits & ((need == 0) | (upto <= count)) & (q_end <= rows)
    taken = torch.where(served, need, 0)
    left = count - torch.where(served & (need > 0), upto, 0).amax()
    # Tokens, row by row.
    q_begin = torch.cat((q_end.new_zeros(1), q_end))
    at = torch.arange(rows, device="cuda")
    request = torch.searchsorted(q_end, at, right=True).clamp_max(requests - 1)
    there = (at < q_end[-1]) & served[request]
    pos = torch.where(there, at - q_begin[request] + cached[request], 0)
    block = pos // page
    behind = (upto - need)[request] + block - had[request]  # how many pages are taken before this one
    fetched = free[(count - 1 - behind).clamp(0, pages - 1)]
    new = there & (block >= had[request])
    page_of = torch.where(new, fetched, table[request, block.clamp_max(width - 1)])
    flat = torch.cat((table.flatten(), table.new_empty(1)))
    flat[torch.where(new, request * width + block, requests * width)] = page_of
    table = flat[:-1].view(requests, width)
    slot = torch.where(there, page_of.long() * page + pos % page, -1)
    k_len = torch.where(served, cached + fresh, 0)
    stored = torch.where(served, cached + fresh, cached)
    out = {"free_left": left.view(1), "stored": stored, "k_len": k_len, "q_begin": q_begin, "slot": slot, "position": pos,
           "unserved": (~served).sum().view(1)}
    return {"table": table, "free": free, **{k: v.to(torch.int32) for k, v in out.items()}}


def _plain_append(state):
    page, pages = state["page"], state["pages"]
    slot = state["slot"].long()
    where = torch.where((slot >= 0) & (slot < pages * page), slot, pages * page)
    new = torch.zeros(pages * page + 1, dtype=torch.bool, device="cuda")
    new[where] = True
    new = new[:-1].view(pages, page)
    first = torch.where(new, torch.arange(page, device="cuda"), page).amin(1)  # tokens before it stay
    old = (torch.arange(page, device="cuda") < first.unsqueeze(1)) & (first < page).unsqueeze(1)

    def rewritten(rows, kept, scale, values):
        """rows [tokens][heads][dim]; kept: the pages' bytes as [pages][heads][token][dim]."""
        heads, dim = rows.shape[1:]
        dense = torch.zeros(pages * page + 1, heads, dim, device="cuda")
        dense[where] = rows.float()
        dense = dense[:-1].view(pages, page, heads, dim).permute(0, 2, 1, 3)
        e = _exponents(dense.abs().amax((2, 3)))
        had = torch.frexp(scale)[1] - 1
        e = torch.where((first > 0).unsqueeze(1), torch.maximum(e, had), e)
        e = torch.where((first < page).unsqueeze(1), e, had)
        stay = kept.float() * _power((had - e).clamp_min(-126)).view(pages, heads, 1, 1)
        fresh = (dense * _power(-e).view(pages, heads, 1, 1)).clamp(-TOP, TOP)
        bytes_ = torch.where(new.view(pages, 1, page, 1), fresh, torch.where(old.view(pages, 1, page, 1), stay, kept.float()))
        bytes_ = bytes_.to(torch.float8_e4m3fn)
        return (bytes_.transpose(2, 3) if values else bytes_).contiguous(), _power(e)

    k, k_scale = rewritten(state["k_new"], state["k"].view(torch.float8_e4m3fn), state["k_scale"], False)
    v, v_scale = rewritten(state["v_new"], state["v"].view(torch.float8_e4m3fn).transpose(2, 3), state["v_scale"], True)
    return {"k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale}


def _plain_attend(state):
    case, t = state["case"], state["q"].dtype
    h, hk, d, page = case["heads"], case["kv_heads"], case["dim"], state["page"]
    n, group = case["requests"], case["heads"] // case["kv_heads"]
    q_begin, k_len = state["q_begin"].long(), state["k_len"].long()
    q_len = q_begin[1:] - q_begin[:-1]
    blocks = state["table"].clamp_min(0).long()
    # [requests][kv heads][keys][dim], and values, of all pages of a table row
    k = state["k"].view(torch.float8_e4m3fn).float() * state["k_scale"].view(state["pages"], hk, 1, 1)
    k = k[blocks].transpose(1, 2).reshape(n, hk, -1, d)
    v = state["v"].view(torch.float8_e4m3fn).float() * state["v_scale"].view(state["pages"], hk, 1, 1)
    v = v[blocks].permute(0, 2, 1, 4, 3).reshape(n, hk, -1, d)
    j = torch.arange(k.shape[2], device="cuda")
    i = torch.arange(state["most"], device="cuda")
    v = v * (j < k_len.unsqueeze(1)).view(n, 1, -1, 1)
    there = i < q_len.unsqueeze(1)
    row = (q_begin[:-1].unsqueeze(1) + i).clamp_max(state["q"].shape[0] - 1)
    q = state["q"][row].float().view(n, -1, hk, group, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)
    pos = (k_len - q_len).unsqueeze(1) + i
    seen = (j <= pos.unsqueeze(2)).view(n, 1, 1, -1, j.numel())
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(d)).view(n, hk, group, -1, j.numel())
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, hk, -1, j.numel()), v).view(n, hk, group, -1, d)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(n, -1, h)
    return {"out": o.permute(0, 3, 1, 2, 4).reshape(n, -1, h, d)[there].to(t), "lse": lse[there]}


def work(case):
    size = 2 if case.get("precision") == "bf16" else 4
    if case["kind"] == "rotate":
        cells = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": cells * size * (4 if case["train"] else 2) + 4 * case["rows"] + 8 * case["dim"] * (2 if case["train"] else 1),
                "flops": cells * (30 if case["train"] else 10)}
    before, fresh, ended = _lengths(case)
    if case["kind"] == "blocks":
        page = case["page"]
        taken = sum(_pages(b + f, page) - _pages(b, page) for b, f in zip(before, fresh))
        given = sum(_pages(e, page) for e in ended)
        rows = sum(fresh) + sum(fresh) // 8 + 1
        return {"bytes": 20 * len(fresh) + 4 * len(ended) + 8 * rows + 8 * (taken + given) + 16, "flops": 0}
    hk, d = case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        touched = sum(_pages(b + f, case["page"]) - b // case["page"] for b, f in zip(before, fresh))
        return {"bytes": sum(fresh) * (2 * hk * d * (size + 1) + 4) + touched * hk * 16, "flops": sum(fresh) * hk * d * 6}
    h, rows = case["heads"], sum(fresh)
    keys = sum(before) + rows
    held = sum(_pages(b + f, case["page"]) for b, f in zip(before, fresh))
    pairs = sum(f * b + f * (f + 1) // 2 for b, f in zip(before, fresh))
    return {"bytes": 2 * rows * h * d * size + 4 * rows * h + 2 * keys * hk * d + held * (8 * hk + 4), "flops": 4 * d * h * pairs}


def exact(case, seed):
    if case["kind"] == "blocks":
        return None  # whole numbers
    state = _STATES[case["kind"]](case, torch.Generator(device="cuda").manual_seed(seed))
    return {"rotate": _exact_rotate, "append": _exact_append, "attend": _exact_attend}[case["kind"]](case, state)


def _exact_rotate(case, state):
    """By complex numbers, the gradients by differentiating."""
    rot, d = case["rot"], case["dim"]
    out = {}
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), state["position"].double().view(-1, 1, 1) * state["freq"])
    for name in ("q", "k"):
        x = state[name].double().contiguous().requires_grad_(case["train"])
        gamma = state["gamma_" + name].double().requires_grad_(case["train"])
        y = x * gamma / (x.pow(2).sum(-1, keepdim=True) / d + state["eps"]).sqrt()
        if case["pairs"] == "halves":
            z = torch.view_as_complex(torch.stack((y[..., :rot // 2], y[..., rot // 2:rot]), -1)) * turn
            y = torch.cat((z.real, z.imag, y[..., rot:]), -1)
        else:
            z = torch.view_as_complex(y[..., :rot].reshape(*y.shape[:2], rot // 2, 2)) * turn
            y = torch.cat((torch.view_as_real(z).reshape(*y.shape[:2], rot), y[..., rot:]), -1)
        out[name] = y.detach()
        if case["train"]:
            out["d" + name], out["dgamma_" + name] = torch.autograd.grad(y, (x, gamma), state["d" + name].double())
    return out


def _exact_power(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _nearest(x):
    """x in 64 bits to the nearest e4m3 value, ties to the even one."""
    step = _exact_power((x.abs().clamp_min(2.0 ** -6).view(torch.int64) >> 52) - 1023 - 3)
    return (torch.round(x / step) * step).clamp(-TOP, TOP)


def _exact_append(case, state):
    """Page by page, as the definition says."""
    page = state["page"]
    slots = state["slot"].tolist()
    runs = []  # (page, first offset, first row, rows)
    for row, s in enumerate(slots):
        if runs and runs[-1][0] == s // page:
            runs[-1][3] += 1
        else:
            runs.append([s // page, s % page, row, 1])
    out = {}
    for name in ("k", "v"):
        held = state[name].view(torch.float8_e4m3fn).double()
        held = held.transpose(2, 3).contiguous() if name == "v" else held
        scale = state[name + "_scale"].double()
        for at, first, row, count in runs:
            x = state[name + "_new"][row:row + count].double().transpose(0, 1)  # [heads][rows][dim]
            every = torch.arange(LEAST, MOST + 1, device="cuda")
            large = x.abs().amax((1, 2)).unsqueeze(1) > TOP * _exact_power(every)  # these are too small
            need = (LEAST + large.sum(1)).clamp_max(MOST)
            had = torch.round(torch.log2(scale[at])).long()
            e = torch.maximum(need, had) if first else need
            held[at, :, :first] = _nearest(held[at, :, :first] * _exact_power(had - e).view(-1, 1, 1))
            held[at, :, first:first + count] = _nearest(x * _exact_power(-e).view(-1, 1, 1))
            scale[at] = _exact_power(e)
        out[name], out[name + "_scale"] = held.transpose(2, 3) if name == "v" else held, scale
    return out


def _exact_attend(case, state):
    """Request by request and head by head."""
    h, hk, d, page = case["heads"], case["kv_heads"], case["dim"], state["page"]
    begin, lens, table = state["q_begin"].tolist(), state["k_len"].tolist(), state["table"].long()
    out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(state["q"].shape[:2], dtype=torch.float64, device="cuda")
    for r, n in enumerate(lens):
        rows = slice(begin[r], begin[r + 1])
        blocks = table[r, :_pages(n, page)]
        for kv in range(hk):
            heads = slice(kv * (h // hk), (kv + 1) * (h // hk))
            k = state["k"][blocks, kv].view(torch.float8_e4m3fn).double() * state["k_scale"][blocks, kv].double().view(-1, 1, 1)
            v = state["v"][blocks, kv].view(torch.float8_e4m3fn).double() * state["v_scale"][blocks, kv].double().view(-1, 1, 1)
            k, v = k.reshape(-1, d)[:n], v.transpose(1, 2).reshape(-1, d)[:n]
            q = state["q"][rows, heads].double().transpose(0, 1).contiguous()
            x = torch.matmul(q, k.t().contiguous()) / math.sqrt(d)
            late = torch.arange(n, device="cuda") > torch.arange(n - q.shape[1], n, device="cuda").unsqueeze(1)
            x = x.masked_fill(late, -math.inf)
            out[rows, heads] = torch.matmul(torch.softmax(x, -1), v).transpose(0, 1)
            lse[rows, heads] = torch.logsumexp(x, -1).transpose(0, 1)
    return {"out": out, "lse": lse}
