"""Plain segment attention in 64 bits, and how far a correct computation may be from it.

The bounds follow the arithmetic: u is the unit roundoff of FP32 (2^-24), w that of a
weight as a product's operand and t that of storage (2^-8 for bf16, else u).  A score is a sum
of `dim` products, so its error is at most (dim + 8) u sum |q k| scale, plus a few u of its size
for scaling, bias, cap and the difference to the row's log-sum; e is the largest of these.
A weight is then off by 2 e relative, an output by (2 e + w + terms u) sum p |v| + t |out|, and
so on through the gradient's formulas.
"""
import math

import numpy as np
import torch

import gatgpu

HIDDEN = gatgpu.HIDDEN
U, UB = 2.0 ** -24, 2.0 ** -8


class Problem:
    """Inputs of one plan on the GPU, values and gradients by formula, and bounds."""

    def __init__(self, q_len, k_len, heads, kv_heads, dim, precision=gatgpu.BF16, mask=gatgpu.MASK_FULL, prefix=None,
                 bias=gatgpu.BIAS_NONE, buckets=0, cap=0.0, scale=None, seed=0, gap=0, packed=True, hidden=0.1):
        self.q_len, self.k_len, self.heads, self.kv_heads, self.dim = list(q_len), list(k_len), heads, kv_heads, dim
        self.precision, self.mask, self.bias, self.buckets, self.cap = precision, mask, bias, buckets, cap
        self.prefix = [0] * len(q_len) if prefix is None else list(prefix)
        self.scale = dim ** -0.5 if scale is None else scale
        self.t = torch.bfloat16 if precision == gatgpu.BF16 else torch.float32
        g = torch.Generator(device="cuda").manual_seed(seed)
        # `gap` rows that belong to nobody before, between and behind the segments
        self.q_begin = gap + np.cumsum([0] + [n + gap for n in self.q_len])[:-1]
        self.k_begin = gap + np.cumsum([0] + [n + gap for n in self.k_len])[:-1]
        self.nq = gap + sum(self.q_len) + gap * len(self.q_len)
        self.nk = gap + sum(self.k_len) + gap * len(self.k_len)

        def rows(n, h, pad):  # rows of a wider array where `packed`
            return torch.randn(max(n, 1), h + pad, dim, generator=g, device="cuda").to(self.t)[:, :h]

        pad = 1 if packed else 0
        self.q, self.k, self.v = rows(self.nq, heads, pad), rows(self.nk, kv_heads, 2 * pad), rows(self.nk, kv_heads, pad)
        self.dout = rows(self.nq, heads, pad)
        self.table = self.dist = None
        if bias == gatgpu.BIAS_LINEAR:
            self.table = torch.rand(heads, generator=g, device="cuda") * 0.2
        if bias == gatgpu.BIAS_TABLE:
            self.table = torch.randn(heads, buckets, generator=g, device="cuda")
            self.ld = [(n + 15) // 16 * 16 for n in self.k_len]
            self.off = np.cumsum([0] + [a * b for a, b in zip(self.q_len, self.ld)])
            self.dist = torch.randint(0, buckets + 3, (max(16, int(self.off[-1])),), generator=g, device="cuda", dtype=torch.uint8)
            self.dist[torch.rand(self.dist.numel(), generator=g, device="cuda") < hidden] = HIDDEN

    def distances(self, s):
        """The writable [q_len][k_len] distances of segment s."""
        a, b = int(self.off[s]), int(self.off[s + 1])
        return self.dist[a:b].view(self.q_len[s], self.ld[s])[:, :self.k_len[s]]

    def plan(self, ctx):
        return gatgpu.Attention(ctx, self.q_len, self.k_len, heads=self.heads, kv_heads=self.kv_heads, dim=self.dim,
                                precision=self.precision, mask=self.mask,
                                prefix=self.prefix if self.mask == gatgpu.MASK_PREFIX else None, bias=self.bias,
                                buckets=self.buckets, scale=self.scale, cap=self.cap, q_begin=self.q_begin,
                                k_begin=self.k_begin)

    def buffers(self, train=True, rest=True):
        """(outputs filled with a sentinel, the call's arrays)."""
        out = {"out": torch.full((max(self.nq, 1), self.heads, self.dim), 7.0, dtype=self.t, device="cuda"),
               "lse": torch.full((max(self.nq, 1), self.heads), 7.0, device="cuda")}
        io = gatgpu.AttentionIO(q=self.q.data_ptr(), k=self.k.data_ptr(), v=self.v.data_ptr(), q_stride=self.q.stride(0),
                                k_stride=self.k.stride(0), v_stride=self.v.stride(0), out=out["out"].data_ptr(),
                                out_stride=out["out"].stride(0), lse=out["lse"].data_ptr())
        if self.table is not None:
            io.bias = self.table.data_ptr()
        if self.dist is not None:
            io.dist = self.dist.data_ptr()
        if train:
            grads = torch.full((max(self.nq, self.nk, 1), self.heads + 2 * self.kv_heads, self.dim), 7.0, dtype=self.t, device="cuda")
            out["dq"] = grads[:max(self.nq, 1), :self.heads]
            out["dk"] = grads[:max(self.nk, 1), self.heads:self.heads + self.kv_heads]
            out["dv"] = grads[:max(self.nk, 1), self.heads + self.kv_heads:]
            io.dout, io.dout_stride = self.dout.data_ptr(), self.dout.stride(0)
            io.dq, io.dk, io.dv = (out[n].data_ptr() for n in ("dq", "dk", "dv"))
            io.dq_stride = io.dk_stride = io.dv_stride = grads.stride(0)
            if self.bias == gatgpu.BIAS_TABLE:
                out["dbias"] = torch.full_like(self.table, 7.0)
                io.dbias = out["dbias"].data_ptr()
            if self.precision == gatgpu.BF16 and rest:
                out["rest"] = torch.full_like(out["out"], 7.0)
                io.rest = out["rest"].data_ptr()
        return out, io

    def run(self, ctx, train=True):
        with self.plan(ctx) as plan:
            out, io = self.buffers(train)
            ws = torch.empty(max(1, plan.workspace_bytes(), plan.workspace_bytes(backward=True)), dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
            plan.forward(io, ws.data_ptr(), ws.numel())
            if train:
                plan.backward(io, ws.data_ptr(), ws.numel())
            ctx.synchronize()
        return out

    def segment(self, s, h, x=None):
        """Segment s, head h in 64 bits: scores before the softmax, what is seen, the capped part's slope and its inputs."""
        x = x or {}
        kv = h // (self.heads // self.kv_heads)
        qa, ka, nq, nk = int(self.q_begin[s]), int(self.k_begin[s]), self.q_len[s], self.k_len[s]
        q = x.get("q", self.q)[qa:qa + nq, h].double()
        k, v = (x.get(n, getattr(self, n))[ka:ka + nk, kv].double() for n in ("k", "v"))
        raw = torch.matmul(q, k.t().contiguous()) * self.scale
        tanh = torch.tanh(raw / self.cap) if self.cap else torch.zeros_like(raw)
        y = self.cap * tanh if self.cap else raw
        i = torch.arange(nq, device="cuda").view(-1, 1) + (nk - nq)
        j = torch.arange(nk, device="cuda").view(1, -1)
        seen = torch.ones(nq, nk, dtype=torch.bool, device="cuda")
        if self.mask == gatgpu.MASK_PREFIX:
            seen = (j <= i) | (j < self.prefix[s])
        dist = None
        table = x.get("table", self.table)
        if self.bias == gatgpu.BIAS_LINEAR:
            y = y - table[h].double() * (i - j).abs()
        if self.bias == gatgpu.BIAS_TABLE:
            dist = self.distances(s).long()
            seen = seen & (dist != HIDDEN)
            dist = dist.clamp_max(self.buckets - 1)
            b = table[h].double()
            y = y + torch.where(b <= -1e6, torch.full_like(b, -math.inf), b)[dist]
        return dict(q=q, k=k, v=v, s=y.masked_fill(~seen, -math.inf), tanh=tanh, dist=dist, qa=qa, ka=ka, nq=nq, nk=nk, kv=kv)

    def weights(self, a):
        top = a["s"].amax(1, keepdim=True) if a["nk"] else a["s"].new_full((a["nq"], 1), -math.inf)
        ref = torch.where(top == -math.inf, torch.zeros_like(top), top)
        e = torch.exp(a["s"] - ref)
        total = e.sum(1, keepdim=True)
        p = e / torch.where(total == 0, torch.ones_like(total), total)
        p = torch.where(a["s"] == -math.inf, torch.zeros_like(p), p)
        lse = torch.where(total == 0, torch.full_like(total, -math.inf), ref + torch.log(total)).squeeze(1)
        return p, lse

    @staticmethod
    def _only(p, x):
        """p @ x with nothing from entries of weight 0, whatever x holds."""
        if bool(torch.isfinite(x).all()):
            return torch.matmul(p, x)
        return torch.where((p == 0).unsqueeze(2), torch.zeros((), dtype=x.dtype, device=x.device), p.unsqueeze(2) * x).sum(1)

    def reference(self, train=True):
        """(values, bounds) of every output in 64 bits."""
        z = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")  # noqa: E731
        h, hk, d = self.heads, self.kv_heads, self.dim
        val = {"out": z(max(self.nq, 1), h, d), "lse": z(max(self.nq, 1), h)}
        if train:
            val.update(dq=z(max(self.nq, 1), h, d), dk=z(max(self.nk, 1), hk, d), dv=z(max(self.nk, 1), hk, d))
            if self.bias == gatgpu.BIAS_TABLE:
                val["dbias"] = z(h, self.buckets)
        tol = {n: torch.zeros_like(x) for n, x in val.items()}
        bf16 = self.precision == gatgpu.BF16
        w, t = (UB, UB) if bf16 else (U, U)
        for s in range(len(self.q_len)):
            for head in range(h):
                a = self.segment(s, head)
                q, k, v, nq, nk, kv = a["q"], a["k"], a["v"], a["nq"], a["nk"], a["kv"]
                if nq == 0:
                    continue
                qs, ks = slice(a["qa"], a["qa"] + nq), slice(a["ka"], a["ka"] + nk)
                p, lse = self.weights(a)
                o = self._only(p, v)
                fin = lambda x: torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)  # noqa: E731
                size = fin(a["s"]).abs().amax().item() if nk else 0.0
                size += fin(lse).abs().max().item()
                reach = (torch.matmul(fin(q).abs(), fin(k).abs().t().contiguous()) * self.scale).amax().item() if nk else 0.0
                e = (d + 8) * U * reach + 6 * U * size + 8 * U * self.cap + 4 * U
                va, da = fin(v).abs(), fin(self.dout[qs, head].double()).abs()
                val["out"][qs, head], val["lse"][qs, head] = o, lse
                tol["out"][qs, head] = (2 * e + w + (nk + 8) * U) * torch.matmul(p, va) + t * o.abs()
                tol["lse"][qs, head] = 2 * e + (nk + 8) * U + 4 * U * size
                if not train or nk == 0:
                    continue
                do = self.dout[qs, head].double()
                dead = lse == -math.inf
                do = torch.where(dead.view(-1, 1), torch.zeros_like(do), do)
                delta = (do * o).sum(1, keepdim=True)
                dp = torch.matmul(do, v.t().contiguous())
                ds = torch.where(p == 0, torch.zeros_like(p), p * (dp - delta))
                dx = ds * (1 - a["tanh"] ** 2) if self.cap else ds
                val["dq"][qs, head] = self._only(dx, k) * self.scale
                val["dk"][ks, kv] += self._only(dx.t().contiguous(), q) * self.scale
                val["dv"][ks, kv] += self._only(p.t().contiguous(), do)
                # delta from the stored output and what rounding took from it (bf16: to 2^-16), itself off by tol[out]
                off_out = (2 * e + w + (nk + 8) * U) * torch.matmul(p, va) + (UB * UB if bf16 else U) * o.abs()
                off_delta = (da * off_out).sum(1, keepdim=True) + (d + 4) * U * (da * fin(o).abs()).sum(1, keepdim=True)
                off_dp = (d + 4) * U * torch.matmul(da, va.t().contiguous())
                pa = fin(p)
                off_ds = pa * ((2 * e + 12 * U) * (fin(dp).abs() + fin(delta).abs()) + off_dp + off_delta)
                off_dx = off_ds + fin(dx).abs() * w
                terms = (max(nq * (h // hk), nk) + 8) * U
                tol["dq"][qs, head] = self.scale * torch.matmul(off_dx + terms * fin(dx).abs(), fin(k).abs()) + t * val["dq"][qs, head].abs()
                tol["dk"][ks, kv] += self.scale * torch.matmul((off_dx + terms * fin(dx).abs()).t().contiguous(), fin(q).abs())
                tol["dv"][ks, kv] += (2 * e + w + terms) * torch.matmul(pa.t().contiguous(), da)
                if self.bias == gatgpu.BIAS_TABLE:
                    # the table's gradient comes from FP32 weights and delta: out's own error is that of its bf16 weights,
                    # which delta shares, and what rest leaves
                    cells = (off_ds + nq * nk * U * ds.abs()).reshape(-1)
                    val["dbias"][head].index_add_(0, a["dist"].reshape(-1), ds.reshape(-1))
                    tol["dbias"][head].index_add_(0, a["dist"].reshape(-1), cells)
        if train:
            for n in ("dk", "dv"):
                tol[n] += t * val[n].abs()
        return val, tol

    def check(self, got, train=True):
        val, tol = self.reference(train)
        qrows = torch.zeros(max(self.nq, 1), dtype=torch.bool, device="cuda")
        krows = torch.zeros(max(self.nk, 1), dtype=torch.bool, device="cuda")
        for b, n in zip(self.q_begin, self.q_len):
            qrows[int(b):int(b) + n] = True
        for b, n in zip(self.k_begin, self.k_len):
            krows[int(b):int(b) + n] = True
        for name, want in val.items():
            rows = None if name == "dbias" else krows if name in ("dk", "dv") else qrows
            have = got[name].double()
            if rows is not None:
                assert bool((have[~rows] == 7.0).all()), f"{name}: rows of no segment were written"
                have, want, off = have[rows], want[rows], tol[name][rows]
            else:
                off = tol[name]
            if not have.numel():
                continue
            fine = torch.isfinite(want)
            assert bool((torch.isfinite(have) == fine).all()), f"{name}: finite where it should not be, or the reverse"
            assert bool((have[want == -math.inf] == -math.inf).all()), name
            far = ((have - want).abs() / (off + 1e-30))[fine]
            worst = float(far.max()) if far.numel() else 0.0
            assert worst <= 1.0, f"{name}: {worst:.3g} times the bound"
