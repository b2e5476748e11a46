"""Segment attention and layer norm, as measurable cases.

Two operators, each with its gradient, stand beside the framework's attention over graph edges:

* ``gatgpu_attention_forward`` / ``_backward``: softmax attention among the rows of each segment (a graph
  or document of a packed batch, or one sequence with its cached keys), with capped scores, a bias by
  distance, a causal mask with a visible prefix, and key/value heads shared by several query heads.
* ``gatgpu_norm_forward`` / ``_backward``: layer norm of a residual sum, optionally followed by ELU, with
  the gradients of its weights.

A case of kind ``attention`` draws its segments' lengths from the case alone (``lengths`` seeds them), so
that its work does not depend on the inputs' seed.  ``run`` is one forward, or, with ``train``, one
forward and one backward on a given output gradient.
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
HIDDEN = 255  # distance of a pair that does not see each other


def _attention(name, segments, lo, hi, heads, kv_heads, dim, precision, train, mask="full", bias="none", buckets=0,
               cap=0.0, queries=0, lengths=1):
    """queries 0: every row of a segment is a query and a key; else that many queries at each segment's end."""
    return {"name": name, "kind": "attention", "segments": segments, "lo": lo, "hi": hi, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "precision": precision, "train": train, "mask": mask, "bias": bias,
            "buckets": buckets, "cap": cap, "queries": queries, "lengths": lengths}


def _norm(name, rows, width, precision, train, residual, elu):
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "precision": precision, "train": train,
            "residual": residual, "elu": elu}


def listed():
    return [
        # One new token of one sequence over its cached keys: the smallest call of a serving loop.
        _attention("attend_token_900", 1, 900, 900, 8, 8, 64, "bf16", False, mask="prefix", bias="linear", queries=1),
        # One new token of each of 48 sequences of very different lengths, key/value heads shared by four.
        _attention("attend_tokens_48x24k", 48, 200, 24_000, 32, 8, 128, "bf16", False, mask="prefix", queries=1),
        # Molecule-sized graphs in a packed batch, shortest-path biases, the model's 8 heads of 32: prediction ...
        _attention("attend_molecules_fwd", 4096, 9, 60, 8, 8, 32, "bf16", False, bias="table", buckets=20),
        # ... and training, in both precisions.
        _attention("attend_molecules_train", 1500, 9, 60, 8, 8, 32, "bf16", True, bias="table", buckets=20),
        _attention("attend_molecules_train_fp32", 500, 9, 60, 4, 4, 16, "fp32", True, bias="table", buckets=12),
        # Graphs of hundreds of nodes, 8 heads of 64, trained with a bias table.
        _attention("attend_graphs_train", 24, 130, 1300, 8, 8, 64, "bf16", True, bias="table", buckets=32),
        # All nodes of one graph, capped scores.
        _attention("attend_all_nodes_16k", 1, 16_384, 16_384, 8, 8, 64, "bf16", False, cap=30.0),
        # Long sequences with a visible prefix, shared key/value heads, capped scores: a training step.
        _attention("attend_prefix_train_4k", 4, 3800, 4400, 16, 4, 128, "bf16", True, mask="prefix", bias="linear",
                   cap=50.0),
        # The rows of one small request.
        _norm("norm_32x256", 32, 256, "fp32", False, False, True),
        # The hidden rows of the 169K-node graph, a training step with residual and ELU.
        _norm("norm_train_169k_256", 169_343, 256, "bf16", True, True, True),
        # An odd narrow width in FP32, a training step.
        _norm("norm_train_50k_100_fp32", 50_021, 100, "fp32", True, False, False),
        # Wide rows, a training step with residual.
        _norm("norm_train_8k_8192", 8_190, 8192, "bf16", True, True, False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    precision = rng.choice(("bf16", "bf16", "bf16", "fp32"))
    if rng.random() < 0.35:
        width = _log_int(rng, 16, 12_000)
        rows = _log_int(rng, 1, min(200_000, 60_000_000 // width))
        return {"kind": "norm", "rows": rows, "width": width, "precision": precision, "train": rng.random() < 0.6,
                "residual": rng.random() < 0.5, "elu": rng.random() < 0.5}
    kv_heads, group = rng.choice(((8, 1), (8, 1), (4, 1), (4, 4), (2, 4), (1, 8), (3, 2)))
    dim = rng.choice((16, 32, 32, 40, 64, 64, 96, 128))
    cap = rng.choice((0.0, 0.0, 30.0, 50.0))
    if rng.random() < 0.25:  # few new rows over cached keys
        hi = _log_int(rng, 100, 20_000)
        return {"kind": "attention", "segments": _log_int(rng, 1, max(2, min(64, 400_000 // hi))),
                "lo": max(1, hi // rng.choice((1, 2, 20))), "hi": hi, "heads": kv_heads * group, "kv_heads": kv_heads,
                "dim": dim, "precision": precision, "train": False, "mask": "prefix",
                "bias": rng.choice(("none", "linear")), "buckets": 0, "cap": cap, "queries": rng.choice((1, 1, 1, 3, 9)),
                "lengths": rng.randrange(1 << 20)}
    hi = _log_int(rng, 12, 4000)
    lo = max(1, hi // rng.choice((1, 2, 6, 12)))
    train = rng.random() < 0.6
    most = (8_000_000_000 if precision == "bf16" else 1_600_000_000) // (kv_heads * group * max(dim, 32)) // (3 if train else 1)
    segments = _log_int(rng, 1, max(1, min(3000, 100_000 // hi, most // (hi * hi))))
    bias = rng.choice(("none", "linear", "table", "table"))
    return {"kind": "attention", "segments": segments, "lo": lo, "hi": hi, "heads": kv_heads * group,
            "kv_heads": kv_heads, "dim": dim, "precision": precision, "train": train,
            "mask": rng.choice(("full", "full", "prefix")), "bias": bias,
            "buckets": rng.randint(4, 64) if bias == "table" else 0, "cap": cap, "queries": 0,
            "lengths": rng.randrange(1 << 20)}


def _lengths(case):
    """Per segment: queries, keys, visible prefix."""
    rng = random.Random(case["lengths"])
    keys = [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["segments"])]
    queries = [min(case["queries"], k) if case["queries"] else k for k in keys]
    prefix = [k // 4 if case["mask"] == "prefix" and not case["queries"] else 0 for k in keys]
    return queries, keys, prefix


def _rows(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0)


def _attention_state(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPE[case["precision"]]
    queries, keys, prefix = _lengths(case)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    nq, nk = sum(queries), sum(keys)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(t)

    state = {"case": case, "queries": queries, "keys": keys, "prefix": prefix, "q_off": _rows(queries).cuda(),
             "k_off": _rows(keys).cuda()}
    if case["queries"]:  # the cache, and the new tokens' queries
        state["q"], kv = normal(nq, h, d), normal(nk, 2 * hk, d)
        state["k"], state["v"] = kv[:, :hk], kv[:, hk:]
    else:  # one projection's rows
        qkv = normal(nk, h + 2 * hk, d)
        state["q"], state["k"], state["v"] = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    if case["train"]:
        state["dout"] = normal(nq, h, d)
    if case["bias"] == "linear":
        state["bias"] = torch.pow(2.0, -8.0 * torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / h)
    if case["bias"] == "table":
        state["bias"] = torch.randn(h, case["buckets"], generator=g, device="cuda")
        # Rows of each segment's distances start at multiples of 16 bytes.
        k = torch.tensor(keys, device="cuda")
        ld = (k + 15) // 16 * 16
        size = torch.tensor(queries, device="cuda") * ld
        state["dist_ld"], state["dist_off"] = ld, size.cumsum(0) - size
        far = -torch.log(torch.rand(int(size.sum()), generator=g, device="cuda").clamp_min(1e-9)) * (case["buckets"] / 3)
        dist = (1 + far).clamp_max(case["buckets"] + 2).to(torch.uint8)
        dist[far > 2.8 * case["buckets"] / 3] = HIDDEN  # about 6 of 100 pairs have no path
        seg = torch.repeat_interleave(torch.arange(len(keys), device="cuda"), torch.tensor(queries, device="cuda"))
        i = torch.arange(nq, device="cuda") - state["q_off"][seg]
        dist[state["dist_off"][seg] + i * ld[seg] + i] = 0
        state["dist"] = dist
    return state


_context = None


def _own_attention(state):
    """The plan, output buffers and workspace that a program keeps."""
    global _context
    import gatgpu

    case, t = state["case"], DTYPE[state["case"]["precision"]]
    if _context is None:
        _context = gatgpu.Context(0)
    plan = gatgpu.Attention(
        _context, state["queries"], state["keys"], heads=case["heads"], kv_heads=case["kv_heads"], dim=case["dim"],
        precision=gatgpu.BF16 if case["precision"] == "bf16" else gatgpu.FP32,
        mask=gatgpu.MASK_PREFIX if case["mask"] == "prefix" else gatgpu.MASK_FULL,
        prefix=state["prefix"] if case["mask"] == "prefix" else None,
        bias={"none": gatgpu.BIAS_NONE, "linear": gatgpu.BIAS_LINEAR, "table": gatgpu.BIAS_TABLE}[case["bias"]],
        buckets=case["buckets"], cap=case["cap"])
    q, k, v = state["q"], state["k"], state["v"]
    out = {"out": torch.empty(q.shape, dtype=t, device="cuda"),
           "lse": torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")}
    io = gatgpu.AttentionIO(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_stride=q.stride(0), k_stride=k.stride(0),
                            v_stride=v.stride(0), out=out["out"].data_ptr(), out_stride=out["out"].stride(0),
                            lse=out["lse"].data_ptr())
    if "bias" in state:
        io.bias = state["bias"].data_ptr()
    if "dist" in state:
        io.dist = state["dist"].data_ptr()
    if case["train"]:
        h, hk = case["heads"], case["kv_heads"]
        grads = torch.empty(k.shape[0], h + 2 * hk, case["dim"], dtype=t, device="cuda")
        out["dq"], out["dk"], out["dv"] = grads[:, :h], grads[:, h:h + hk], grads[:, h + hk:]
        io.dout, io.dout_stride = state["dout"].data_ptr(), state["dout"].stride(0)
        io.dq, io.dk, io.dv = (out[n].data_ptr() for n in ("dq", "dk", "dv"))
        io.dq_stride = io.dk_stride = io.dv_stride = grads.stride(0)
        if case["bias"] == "table":
            out["dbias"] = torch.empty_like(state["bias"])
            io.dbias = out["dbias"].data_ptr()
        if case["precision"] == "bf16":  # what rounding took from out: the gradients keep their precision
            state["rest"] = torch.empty_like(out["out"])
            io.rest = state["rest"].data_ptr()
    need = max(plan.workspace_bytes(), plan.workspace_bytes(backward=True) if case["train"] else 0)
    state["work"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    state.update(plan=plan, io=io, outputs=out)


def _norm_state(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPE[case["precision"]]
    rows, width = case["rows"], case["width"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    state = {"case": case, "x": (normal(rows, width) * 1.5 + 0.3).to(t), "gamma": 1 + 0.2 * normal(width),
             "beta": 0.2 * normal(width), "eps": 1e-5}
    if case["residual"]:
        state["residual"] = normal(rows, width).to(t)
    if case["train"]:
        state["dy"] = normal(rows, width).to(t)
        if case["residual"]:
            state["dsum"] = normal(rows, width).to(t)
    return state


def _own_norm(state):
    global _context
    import gatgpu

    case, x = state["case"], state["x"]
    if _context is None:
        _context = gatgpu.Context(0)
    rows, width = x.shape
    out = {"y": torch.empty_like(x)}
    io = gatgpu.NormIO(precision=gatgpu.BF16 if case["precision"] == "bf16" else gatgpu.FP32, elu=int(case["elu"]),
                       rows=rows, width=width, eps=state["eps"], x=x.data_ptr(), x_stride=width,
                       gamma=state["gamma"].data_ptr(), beta=state["beta"].data_ptr(), y=out["y"].data_ptr(),
                       y_stride=width)
    if case["residual"]:
        out["sum"] = torch.empty_like(x)
        io.residual, io.residual_stride = state["residual"].data_ptr(), width
        io.sum, io.sum_stride = out["sum"].data_ptr(), width
    if case["train"]:
        for name in ("mean", "rstd"):
            out[name] = torch.empty(rows, dtype=torch.float32, device="cuda")
        for name in ("dgamma", "dbeta"):
            out[name] = torch.empty(width, dtype=torch.float32, device="cuda")
        out["dx"] = torch.empty_like(x)
        io.mean, io.rstd = out["mean"].data_ptr(), out["rstd"].data_ptr()
        io.dy, io.dy_stride = state["dy"].data_ptr(), width
        io.dx, io.dx_stride = out["dx"].data_ptr(), width
        io.dgamma, io.dbeta = out["dgamma"].data_ptr(), out["dbeta"].data_ptr()
        if case["residual"]:
            io.dsum, io.dsum_stride = state["dsum"].data_ptr(), width
        state["work"] = torch.empty(max(1, _context.norm_workspace(rows, width)), dtype=torch.uint8, device="cuda")
    state.update(io=io, outputs=out)


def prepare(case, seed):
    if case["kind"] == "norm":
        state = _norm_state(case, seed)
        if own:
            _own_norm(state)
    else:
        state = _attention_state(case, seed)
        if own:
            _own_attention(state)
    return state


def run(state):
    case = state["case"]
    if own:
        work = state.get("work")
        if case["kind"] == "norm":
            _context.norm_forward(state["io"])
            if case["train"]:
                _context.norm_backward(state["io"], work.data_ptr(), work.numel())
        else:
            state["plan"].forward(state["io"], work.data_ptr(), work.numel())
            if case["train"]:
                state["plan"].backward(state["io"], work.data_ptr(), work.numel())
        return state["outputs"]
    return _plain_norm(state) if case["kind"] == "norm" else _plain_attention(state)


def _plain_norm(state):
    case, t = state["case"], state["x"].dtype
    h = state["x"].float()
    out = {}
    if case["residual"]:
        out["sum"] = (h + state["residual"].float()).to(t)
        h = out["sum"].float()  # the norm is that of the stored rows
    mean = h.mean(1, keepdim=True)
    rstd = torch.rsqrt((h - mean).square().mean(1, keepdim=True) + state["eps"])
    n = (h - mean) * rstd
    pre = n * state["gamma"] + state["beta"]
    out["y"] = (torch.where(pre > 0, pre, torch.expm1(pre)) if case["elu"] else pre).to(t)
    if case["train"]:
        dt = state["dy"].float()
        if case["elu"]:
            dt = torch.where(pre > 0, dt, dt * torch.exp(pre))
        out["mean"], out["rstd"] = mean.squeeze(1), rstd.squeeze(1)
        out["dgamma"] = (dt * n).sum(0, dtype=torch.float64).float()
        out["dbeta"] = dt.sum(0, dtype=torch.float64).float()
        dn = dt * state["gamma"]
        dx = rstd * (dn - dn.mean(1, keepdim=True) - n * (dn * n).mean(1, keepdim=True))
        if case["residual"]:
            dx = dx + state["dsum"].float()
        out["dx"] = dx.to(t)
    return out


def _padded(rows, off, longest):
    """[segments][longest][...] of packed rows, zero behind each segment's end, and which of them are rows."""
    at = torch.arange(longest, device=rows.device)
    there = at < (off[1:] - off[:-1]).unsqueeze(1)
    index = (off[:-1].unsqueeze(1) + at).clamp_max(rows.shape[0] - 1)
    full = rows[index].float()
    return full * there.view(*there.shape, *([1] * (rows.dim() - 1))), there


def _plain_attention(state):
    case, t = state["case"], state["q"].dtype
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    scale, cap = 1.0 / math.sqrt(d), case["cap"]
    segments, lq, lk = len(state["keys"]), max(state["queries"]), max(state["keys"])
    q, q_there = _padded(state["q"], state["q_off"], lq)
    k, k_there = _padded(state["k"], state["k_off"], lk)
    v, _ = _padded(state["v"], state["k_off"], lk)
    # [segments][kv heads][group * queries][dim]: the query heads that share a key/value head side by side
    q = q.view(segments, lq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(segments, hk, -1, d)
    k, v = (x.permute(0, 2, 1, 3).contiguous() for x in (k, v))
    nq, nk = (off[1:] - off[:-1] for off in (state["q_off"], state["k_off"]))
    i, j = torch.arange(lq, device="cuda"), torch.arange(lk, device="cuda")
    there = (q_there.unsqueeze(2) & k_there.unsqueeze(1))  # [segments][lq][lk]
    pos = i + (nk - nq).unsqueeze(1)
    if case["mask"] == "prefix":
        prefix = torch.tensor(state["prefix"], device="cuda").view(-1, 1, 1)
        there &= (j <= pos.unsqueeze(2)) | (j < prefix)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(scale).view(segments, hk, h // hk, lq, lk)
    if cap:
        score = torch.tanh(score.div_(cap)).mul_(cap)
        slope = 1 - (score / cap).square() if case["train"] else None
    if case["bias"] == "linear":
        score -= state["bias"].view(1, hk, h // hk, 1, 1) * (pos.unsqueeze(2) - j).abs().view(segments, 1, 1, lq, lk)
    if case["bias"] == "table":
        at = state["dist_off"].view(-1, 1, 1) + i.view(-1, 1) * state["dist_ld"].view(-1, 1, 1) + j
        dist = state["dist"][at.clamp_max_(state["dist"].numel() - 1)].long()
        del at
        there &= dist != HIDDEN
        dist.clamp_max_(case["buckets"] - 1)
        score += state["bias"][:, dist].view(hk, h // hk, segments, lq, lk).permute(2, 0, 1, 3, 4)
    there = there.view(segments, 1, 1, lq, lk)
    score.masked_fill_(~there, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    o = torch.matmul(p.view(segments, hk, -1, lk), v)

    def packed(x, off, there, heads):
        """[segments][kv heads][group * rows][dim] back to rows [n][heads][dim] of type t."""
        x = x.view(segments, hk, heads // hk, -1, d).permute(0, 3, 1, 2, 4).reshape(segments, -1, heads, d)
        return x[there].to(t)

    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(segments, lq, h)
    out = {"out": packed(o, state["q_off"], q_there, h), "lse": lse[q_there]}
    if not case["train"]:
        return out
    do, _ = _padded(state["dout"], state["q_off"], lq)
    do = do.view(segments, lq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(segments, hk, -1, d)
    p = p.view(segments, hk, -1, lk)
    out["dv"] = packed(torch.matmul(p.transpose(2, 3), do), state["k_off"], k_there, hk)
    ds = torch.matmul(do, v.transpose(2, 3)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if case["bias"] == "table":
        each = ds.view(segments, h, lq, lk)
        out["dbias"] = torch.stack([torch.where((dist == b).unsqueeze(1), each, 0).sum((0, 2, 3), dtype=torch.float64)
                                    for b in range(case["buckets"])], 1).float()
    if cap:
        ds.mul_(slope.view(ds.shape))
    ds.mul_(scale)
    out["dq"] = packed(torch.matmul(ds, k), state["q_off"], q_there, h)
    out["dk"] = packed(torch.matmul(ds.transpose(2, 3), q), state["k_off"], k_there, hk)
    return out


def _pairs(case):
    """Query/key pairs that the masks by position leave, over all segments."""
    total = 0
    for nq, nk, prefix in zip(*_lengths(case)):
        if case["mask"] == "full":
            total += nq * nk
        else:
            first = nk - nq + 1  # keys that the first query sees
            total += nq * first + nq * (nq - 1) // 2
            short = max(0, prefix - first)  # the prefix shows more to the queries before it
            total += short * (short + 1) // 2
    return total


def work(case):
    size = 2 if case["precision"] == "bf16" else 4
    if case["kind"] == "norm":
        cells = case["rows"] * case["width"]
        passes = 2 + 2 * case["residual"] + case["train"] * (3 + case["residual"])
        return {"bytes": cells * size * passes + (16 * case["width"] + 8 * case["rows"] if case["train"] else 8 * case["width"]),
                "flops": cells * (8 + 14 * case["train"])}
    queries, keys, _ = _lengths(case)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    qs, ks = sum(queries) * h * d * size, sum(keys) * hk * d * size
    nbytes = 2 * qs + 2 * ks + 4 * sum(queries) * h
    flops = 4 * d * h * _pairs(case)
    if case["bias"] == "table":
        nbytes += sum(a * b for a, b in zip(queries, keys)) + 4 * h * case["buckets"]
    if case["train"]:  # dout read, dq, dk, dv written: what came before stays what it was
        nbytes += 2 * qs + 2 * ks + (4 * h * case["buckets"] if case["bias"] == "table" else 0)
        flops += 10 * d * h * _pairs(case)
    return {"bytes": nbytes, "flops": flops}


def exact(case, seed):
    if case["kind"] == "norm":
        return _exact_norm(_norm_state(case, seed))
    return _exact_attention(_attention_state(case, seed))


def _exact_norm(state):
    case = state["case"]
    out = {}
    h = state["x"].double()
    if case["residual"]:
        h = (h + state["residual"].double()).to(state["x"].dtype).double()
        out["sum"] = h.clone()
    gamma, beta = (state[n].double().requires_grad_(case["train"]) for n in ("gamma", "beta"))
    h.requires_grad_(case["train"])
    centred = h - h.mean(1, keepdim=True)
    spread = (centred.pow(2).mean(1, keepdim=True) + state["eps"]).sqrt()
    y = centred / spread * gamma + beta
    if case["elu"]:
        y = torch.nn.functional.elu(y)
    out["y"] = y.detach()
    if case["train"]:
        y.backward(state["dy"].double())
        out["mean"], out["rstd"] = h.detach().mean(1), 1 / spread.detach().squeeze(1)
        out["dgamma"], out["dbeta"], out["dx"] = gamma.grad, beta.grad, h.grad
        if case["residual"]:
            out["dx"] = out["dx"] + state["dsum"].double()
    return out


def _exact_attention(state):
    """Segment by segment, the gradients by differentiating the definition."""
    case = state["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    queries, keys, prefix = state["queries"], state["keys"], state["prefix"]
    out = {"out": torch.empty(state["q"].shape, dtype=torch.float64, device="cuda"),
           "lse": torch.empty(state["q"].shape[:2], dtype=torch.float64, device="cuda")}
    table = state["bias"].double().requires_grad_(case["train"]) if "bias" in state else None
    if case["train"]:
        for name, like in (("dq", "q"), ("dk", "k"), ("dv", "v")):
            out[name] = torch.empty(state[like].shape, dtype=torch.float64, device="cuda")
        if case["bias"] == "table":
            out["dbias"] = torch.zeros(state["bias"].shape, dtype=torch.float64, device="cuda")
    qa, ka = _rows(queries).tolist(), _rows(keys).tolist()
    heads_at_once = max(1, int(1.5e9 / (max(queries) * max(keys)) / 8))
    where = state["dist_off"].tolist() if "dist" in state else None
    for s in range(len(keys)):
        nq, nk = queries[s], keys[s]
        i, j = torch.arange(nq, device="cuda").view(-1, 1) + (nk - nq), torch.arange(nk, device="cuda").view(1, -1)
        seen = torch.ones(nq, nk, dtype=torch.bool, device="cuda")
        if case["mask"] == "prefix":
            seen = (j <= i) | (j < prefix[s])
        if where is not None:
            ld = (nk + 15) // 16 * 16
            dist = state["dist"][where[s]:where[s] + nq * ld].view(nq, ld)[:, :nk].long()
            seen = seen & (dist != HIDDEN)
        for kv in range(hk):
            group = h // hk
            for first in range(kv * group, kv * group + group, heads_at_once):
                hs = slice(first, min(first + heads_at_once, kv * group + group))
                q = state["q"][qa[s]:qa[s + 1], hs].double().transpose(0, 1).contiguous().requires_grad_(case["train"])
                k, v = (state[n][ka[s]:ka[s + 1], kv].double().contiguous().requires_grad_(case["train"]) for n in ("k", "v"))
                x = torch.matmul(q, k.t().contiguous()) / math.sqrt(d)
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if case["bias"] == "linear":
                    x = x - table[hs].view(-1, 1, 1) * (i - j).abs()
                if case["bias"] == "table":
                    x = x + table[hs][:, dist.clamp_max(case["buckets"] - 1)]
                x = x.masked_fill(~seen, -math.inf)
                o = torch.matmul(torch.softmax(x, -1), v)
                out["out"][qa[s]:qa[s + 1], hs] = o.detach().transpose(0, 1)
                out["lse"][qa[s]:qa[s + 1], hs] = torch.logsumexp(x.detach(), -1).transpose(0, 1)
                if not case["train"]:
                    continue
                wanted = [q, k, v] + ([table] if case["bias"] == "table" else [])
                do = state["dout"][qa[s]:qa[s + 1], hs].double().transpose(0, 1).contiguous()
                got = torch.autograd.grad(o, wanted, do)
                out["dq"][qa[s]:qa[s + 1], hs] = got[0].transpose(0, 1)
                for name, value in (("dk", got[1]), ("dv", got[2])):
                    at = out[name][ka[s]:ka[s + 1], kv]
                    at.copy_(value if first == kv * group else at + value)
                if case["bias"] == "table":
                    out["dbias"] += got[3]
    return out
