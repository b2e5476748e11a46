"""Plain forms, in 64 bits, of the paged cache's operators and of norms and rotation of queries and keys."""
import math

import numpy as np
import torch

import gatgpu

TOP, LEAST, MOST = 448.0, -64, 64
EPS = {gatgpu.BF16: 2.0 ** -8, gatgpu.FP32: 2.0 ** -24}  # half a step of the storage, relative
TYPE = {gatgpu.BF16: torch.bfloat16, gatgpu.FP32: torch.float32}


def generator(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g)


# -- e4m3
def values(bytes_):
    """What e4m3 bytes stand for, by the format: sign, 4 bits of exponent (bias 7), 3 of mantissa, 0x7f NaN."""
    b = bytes_.to(torch.int64)
    e, m = (b >> 3) & 15, (b & 7).double()
    x = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.pow(torch.tensor(2.0, dtype=torch.float64), (e - 7).double()))
    x = torch.where((b & 127) == 127, math.nan, x)
    return torch.where(b >= 128, -x, x)


def bytes_of(x):
    """64-bit values to e4m3 bytes: nearest, ties to even; NaN to 0x7f (either sign).  |x| <= 448 but for NaN."""
    a = torch.nan_to_num(x.abs(), nan=0.0)
    e = torch.floor(torch.log2(a.clamp_min(2.0 ** -6)))
    q = torch.round(a * torch.pow(2.0, 3 - e))  # steps of 2^(e - 3), ties to even
    up = q >= 16  # (only where e is exact is q below 16 otherwise)
    e, q = torch.where(up, e + 1, e), torch.where(up, torch.round(q / 2), q)
    code = torch.where(q < 8, q, (e + 6) * 8 + q).to(torch.int64)  # q in [8, 16): exponent field e + 7, mantissa q - 8
    code = torch.where(torch.isnan(x), 127, code)
    return (code + 128 * torch.signbit(x).to(torch.int64)).to(torch.uint8)


def exponent(amax):
    """Least e with amax <= 448 2^e, in the scales' range, by trying each."""
    e = LEAST
    while e < MOST and amax > TOP * 2.0 ** e:
        e += 1
    return e


class Pages:
    """A cache on the host: bytes and scales in the library's layout."""

    def __init__(self, pages, page, heads, dim, seed=0, stale=True):
        g = generator(seed)
        self.pages, self.page, self.heads, self.dim = pages, page, heads, dim
        hi = 256 if stale else 1  # whatever was there before, NaN among it
        self.k = torch.randint(0, hi, (pages, heads, page, dim), generator=g, dtype=torch.uint8)
        self.v = torch.randint(0, hi, (pages, heads, dim, page), generator=g, dtype=torch.uint8)
        self.k_scale = torch.pow(2.0, torch.randint(-9, 3, (pages, heads), generator=g).float())
        self.v_scale = torch.pow(2.0, torch.randint(-9, 3, (pages, heads), generator=g).float())

    def sides(self):
        """(bytes as [page][head][token][dim], scales) of keys and values; both are views."""
        return (self.k, self.k_scale), (self.v.transpose(2, 3), self.v_scale)

    def append(self, k, v, slots):
        """The operator's definition, page by page and head by head."""
        runs, slots = [], slots.tolist()
        for row, s in enumerate(slots):
            if not 0 <= s < self.pages * self.page:
                continue
            if runs and runs[-1][1] == row and s % self.page and slots[row - 1] == s - 1:
                runs[-1][1] += 1
            else:
                runs.append([row, row + 1])
        for (data, scale), new in zip(self.sides(), (k, v)):
            for lo, hi in runs:
                p, off = divmod(slots[lo], self.page)
                for h in range(self.heads):
                    x = new[lo:hi, h].double()
                    fine = x[torch.isfinite(x)].abs()
                    e = exponent(float(fine.max()) if fine.numel() else 0.0)
                    had = int(math.log2(float(scale[p, h])))
                    if off:
                        e = max(e, had)
                        data[p, h, :off] = bytes_of(values(data[p, h, :off]) * 2.0 ** (had - e)) if e > had else data[p, h, :off]
                    x = torch.where(torch.isfinite(x), (x * 2.0 ** -e).clamp(-TOP, TOP), math.nan)
                    data[p, h, off:off + hi - lo] = bytes_of(x)
                    scale[p, h] = 2.0 ** e

    def device(self):
        d = {n: getattr(self, n).cuda() for n in ("k", "v", "k_scale", "v_scale")}
        d["cache"] = gatgpu.Cache(pages=self.pages, page=self.page, kv_heads=self.heads, dim=self.dim, **{n: t.data_ptr() for n, t in d.items()})
        return d

    def same_values(self, d):
        """Bytes on the device stand for the same values (NaNs of either sign are one)."""
        for n in ("k", "v"):
            a, b = values(getattr(self, n)), values(d[n].cpu())
            assert torch.equal(torch.isnan(a), torch.isnan(b)), n
            assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)), n
        assert torch.equal(self.k_scale, d["k_scale"].cpu()) and torch.equal(self.v_scale, d["v_scale"].cpu())


def attention(pages, q, q_begin, k_len, table, scale, most=None):
    """out, lse and a bound's weight per output: [rows][heads][dim], in 64 bits.  Rows of no request: NaN (not written)."""
    rows, heads, dim = q.shape
    out = torch.full((rows, heads, dim), math.nan, dtype=torch.float64)
    lse = torch.full((rows, heads), math.nan, dtype=torch.float64)
    spread = torch.zeros(rows, heads, dim, dtype=torch.float64)  # sum p |v|
    reach = torch.zeros(rows, heads, dtype=torch.float64)        # largest scale sum |q k|
    (kb, ks), (vb, vs) = pages.sides()
    group = heads // pages.heads
    for r, keys in enumerate(k_len):
        lo, hi = q_begin[r], q_begin[r + 1]
        n = min(keys, len(table[r]) * pages.page)
        blocks = [int(b) for b in table[r][:(n + pages.page - 1) // pages.page]]
        held = torch.tensor([0 <= b < pages.pages for b in blocks for _ in range(pages.page)], dtype=torch.bool)[:n]
        use = [b if 0 <= b < pages.pages else 0 for b in blocks]
        for kv in range(pages.heads):
            k = (values(kb[use, kv]) * ks[use, kv].double().view(-1, 1, 1)).reshape(-1, dim)[:n]
            v = (values(vb[use, kv]) * vs[use, kv].double().view(-1, 1, 1)).reshape(-1, dim)[:n]
            for i in range(hi - lo if most is None else min(hi - lo, most)):
                pos = n - (hi - lo) + i
                seen = held & (torch.arange(n) <= pos)
                for h in range(kv * group, (kv + 1) * group):
                    row = q[lo + i, h].double()
                    x = scale * (k[seen] @ row)
                    if not bool((x > -math.inf).any()) and not bool(torch.isnan(x).any()):
                        out[lo + i, h], lse[lo + i, h] = 0.0, -math.inf
                        continue
                    p = torch.softmax(x, 0)
                    out[lo + i, h] = p @ v[seen]
                    lse[lo + i, h] = torch.logsumexp(x, 0)
                    spread[lo + i, h] = p @ v[seen].abs()
                    reach[lo + i, h] = scale * (k[seen].abs() @ row.abs()).max()
    return out, lse, spread, reach


def attention_bounds(precision, spread, reach, keys, want):
    """How far out and lse may be.  A score's product of dim <= 128 terms in FP32, its scaling and the exponent's
    argument (up to reach log2 e, rounded a few times) change a weight by reach * 2^-24 * (128 + 8); FP32 sums of the
    weights and of their products by keys * 2^-24 at most (the tree's depth in fact); the exponential by 2^-22; then the
    result's own rounding.  Weights are rounded to fp16: 11 significant bits, so a step of 2^-10 in [1, 2) and an error of at
    most half of it, torch.finfo(torch.float16).eps / 2 = 2^-11 of the weight; the second fp16 part of FP32 calls rounds that
    rest once more, 2^-11 * 2^-11 = 2^-22."""
    weight = reach * 2.0 ** -24 * 136 + 2.0 ** -21 + min(keys, 4096) * 2.0 ** -24
    fp16 = 2.0 ** -11 if precision == gatgpu.BF16 else 2.0 ** -22
    tol_out = spread * (2 * weight.unsqueeze(-1) + fp16) + want.abs() * EPS[precision] + 1e-30
    tol_lse = weight + 2.0 ** -22
    return tol_out, tol_lse


def check_attention(pages, q, q_begin, k_len, table, scale, precision, got, got_lse, most=None):
    """A call's out and lse, which held 7 before."""
    out, lse, spread, reach = attention(pages, q, q_begin, k_len, table, scale, most)
    ours = torch.zeros(q.shape[0], dtype=torch.bool)  # rows that are written
    for lo, hi in zip(q_begin, q_begin[1:]):
        ours[lo:hi if most is None else min(hi, lo + most)] = True
    assert bool((got[~ours] == 7).all()) and bool((got_lse[~ours] == 7).all())
    got, got_lse, out, lse, spread, reach = (x[ours].double() for x in (got, got_lse, out, lse, spread, reach))
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    tol_out, tol_lse = attention_bounds(precision, spread, reach, max(k_len), out)
    fine = ~torch.isnan(out)
    err = ((got - out).abs() / tol_out)[fine]
    assert err.numel() == 0 or float(err.max()) <= 1, float(err.max())
    empty = lse == -math.inf
    assert torch.equal(got_lse == -math.inf, empty) and bool((got[empty] == 0).all())
    fine = ~empty & ~torch.isnan(lse)
    err = ((got_lse - lse).abs() / tol_lse)[fine]
    assert err.numel() == 0 or float(err.max()) <= 1, float(err.max())


# -- calls on the GPU
def words(values):
    return torch.from_numpy(np.asarray(list(values), np.uint64).astype(np.uint32).view(np.int32)).cuda()


class Serving:
    """A cache with whatever bytes, and a packed batch of queries over it."""

    def __init__(self, k_len, q_len, heads, kv_heads, dim, page, precision, seed=0, extra_rows=0, stride=0, size=1.0):
        g = generator(seed)
        need = [-(-k // page) for k in k_len]
        self.blocks = max(need + [1])
        self.host = Pages(sum(need) + 2, page, kv_heads, dim, seed=seed + 1)
        order = torch.randperm(sum(need) + 2, generator=g).tolist()
        self.table = [[order.pop() for _ in range(n)] + [gatgpu.NO_PAGE] * (self.blocks + stride - n) for n in need]
        for r, n in enumerate(k_len):  # tokens' values; behind them whatever was there
            for (data, scale), s in zip(self.host.sides(), (size, 1.0)):
                for b in range(need[r]):
                    p, count = self.table[r][b], min(page, n - b * page)
                    x = torch.randn(kv_heads, count, dim, generator=g).double() * 100
                    data[p, :, :count] = bytes_of(x.clamp(-448, 448))
                    scale[p] = 2.0 ** torch.randint(-8, -5, (kv_heads,), generator=g).float() * s
        self.k_len, self.q_len, self.precision = list(k_len), list(q_len), precision
        self.q_begin = [0] + np.cumsum(q_len).tolist()
        self.rows = self.q_begin[-1] + extra_rows
        self.q = normal(g, max(1, self.rows), heads, dim).to(TYPE[precision])
        self.heads, self.dim, self.scale, self.most = heads, dim, dim ** -0.5, max(list(q_len) + [1])

    def device(self, gap=0):
        d = self.host.device()
        per = 8 if self.precision == gatgpu.BF16 else 4
        q = torch.full((max(1, self.rows), self.heads * self.dim + gap * per), 3.0, dtype=TYPE[self.precision])
        q[:, :self.heads * self.dim] = self.q.reshape(max(1, self.rows), -1)
        d.update(q=q.cuda(), q_begin=words(self.q_begin), lens=words(self.k_len), table=words([x for row in self.table for x in row]))
        d["out"] = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
        d["lse"] = torch.full((max(1, self.rows), self.heads), 7.0, device="cuda")
        return d

    def io(self, d, **change):
        io = gatgpu.CacheAttentionIO(precision=self.precision, heads=self.heads, scale=self.scale, rows=self.rows, requests=len(self.k_len), most=self.most,
                                     blocks=self.blocks, table_stride=len(self.table[0]), q=d["q"].data_ptr(), q_stride=d["q"].stride(0),
                                     q_begin=d["q_begin"].data_ptr(), k_len=d["lens"].data_ptr(), table=d["table"].data_ptr(), out=d["out"].data_ptr(),
                                     out_stride=d["out"].stride(0), lse=d["lse"].data_ptr())
        for k, v in change.items():
            setattr(io, k, v)
        return io

    def run(self, ctx, gap=1, **change):
        d = self.device(gap)
        io = self.io(d, **change)
        need = ctx.cache_attention_workspace(d["cache"], io)
        work = torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # (NaN, if it were read)
        torch.cuda.synchronize()
        ctx.cache_attention(d["cache"], io, work.data_ptr(), need)
        ctx.synchronize()
        return d

    def check(self, d, most=None):
        wide = self.heads * self.dim
        got, got_lse = d["out"].cpu()[:, :wide].view(-1, self.heads, self.dim)[:self.rows], d["lse"].cpu()[:self.rows]
        assert bool((d["out"][:, wide:] == 7).all())
        check_attention(self.host, self.q[:self.rows], self.q_begin, self.k_len, self.table, self.scale, self.precision, got, got_lse, most)


# -- norms and rotation
def rotate(x, gamma, eps, norm, position, freq, rot, pairs):
    """x [rows][heads][dim] in 64 bits (differentiable)."""
    t = x
    if norm:
        t = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * (gamma if gamma is not None else 1.0)
    if rot:
        angle = position.double().view(-1, 1, 1) * freq
        c, s = torch.cos(angle), torch.sin(angle)
        first = torch.arange(rot // 2) if pairs == gatgpu.PAIRS_HALVES else 2 * torch.arange(rot // 2)
        second = first + (rot // 2 if pairs == gatgpu.PAIRS_HALVES else 1)
        a, b = t[..., first], t[..., second]
        t = t.clone()
        t[..., first] = a * c - b * s
        t[..., second] = b * c + a * s
    return t


# -- block tables
def assign(cached, fresh, table, free, count, page, pages, blocks, rows):
    """One request after another; lists of ints, table rows are changed in place."""
    count = min(count, pages)
    left, total, out = count, 0, {"stored": [], "k_len": [], "q_begin": [0], "slot": [gatgpu.NO_PAGE] * rows, "position": [0] * rows}
    unserved, taken, promised = 0, {}, 0
    for r, (c, f) in enumerate(zip(cached, fresh)):
        fits = c + f <= blocks * page
        need = (c + f + page - 1) // page - (c + page - 1) // page if fits else 0
        promised += need
        total += f
        served = fits and (need == 0 or promised <= count) and total <= rows
        unserved += not served
        if served and need:
            left = min(left, count - promised)
        if served:
            had = (c + page - 1) // page
            for b in range(need):
                table[r][had + b] = free[count - 1 - (promised - need + b)]
            for i in range(f):
                pos = c + i
                p = table[r][pos // page]
                out["position"][total - f + i] = pos
                out["slot"][total - f + i] = p * page + pos % page if 0 <= p < pages else gatgpu.NO_PAGE
        out["stored"].append(c + f if served else c)
        out["k_len"].append(c + f if served else 0)
        out["q_begin"].append(min(total, 2 ** 32 - 1))
    return {**out, "free_left": [left], "unserved": [unserved]}


def release(cached, table, free, count, page, pages, blocks):
    count = min(count, pages)
    for r, c in enumerate(cached):
        for b in range(min((c + page - 1) // page, blocks)):
            if 0 <= table[r][b] < pages:
                if count < pages:
                    free[count] = table[r][b]
                count += 1
    return min(count, pages)


def rotate_bound(x, y, gamma, eps, norm, rot, pairs, precision):
    """How far y = rotate(x) may be off: the norm's factor (a sum of dim squares, a root, a quotient), three products, an angle
    rounded to 2^-25 of a turn, sine and cosine, each relative to the magnitudes of a pair; then y's own rounding."""
    r = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) if norm else torch.ones_like(x[..., :1])
    m = (x * r * (gamma if gamma is not None and norm else 1.0)).abs()
    both = m.clone()
    if rot:
        first = torch.arange(rot // 2) * (1 if pairs == gatgpu.PAIRS_HALVES else 2)
        second = first + (rot // 2 if pairs == gatgpu.PAIRS_HALVES else 1)
        both[..., first] = both[..., second] = m[..., first] + m[..., second]
    rel = (x.shape[-1] / 2 + 12) * 2.0 ** -24 + 2.0 ** -21
    return both * rel + y.abs() * EPS[precision] + 1e-37
