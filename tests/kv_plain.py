"""Plain statements of the operators over the quantized paged cache, on the CPU in 64 bits: attention of
one new token a sequence, with the bound that the kernels' arithmetic allows, and the page pool as
lists."""

from __future__ import annotations

import math

import torch

import mx_plain

CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "mxfp4": torch.uint8}


def empty_cache(kind, pages, page, heads, dim, layout="plain", poison=True):
    """(codes, scales) of one side on the CPU.  `poison`: every slot reads as NaN until it is written."""
    width = dim // 2 if kind == "mxfp4" else dim
    code = {"int8": 0x81, "fp8": 0x7F, "mxfp4": 0x77}[kind] if poison else 0

    def make(last, dtype, fill):
        if layout == "heads_first":  # [pages, heads, page, ...] seen as [pages, page, heads, ...]
            return torch.full((pages, heads, page, last), fill, dtype=dtype).transpose(1, 2)
        if layout == "interleaved":  # one of two sides of every page, with a gap after every head
            return torch.full((pages, 2, page, heads, last + 3), fill, dtype=dtype)[:, 1, :, :, :last]
        return torch.full((pages, page, heads, last), fill, dtype=dtype)

    codes = make(width, torch.uint8, code).view(CODES[kind])
    if kind == "mxfp4":
        return codes, make(dim // 32, torch.uint8, 255 if poison else 0)
    return codes, make(1, torch.float32, math.nan if poison else 0.0)[..., 0]


def put(codes, scales, kind, page, off, x):
    """Writes vectors x [n, heads, dim] to slots (page[n], off[n])."""
    q, s = mx_plain.vector_codes(x, kind)
    codes.view(torch.uint8)[page, off] = q.view(torch.uint8)
    scales[page, off] = s


def vectors(codes, scales, kind, page, off):
    """The values of slots in 64 bits, unrounded: [n, heads, dim]."""
    q, s = codes.view(torch.uint8)[page, off], scales[page, off]
    if kind == "mxfp4":
        return mx_plain.values(mx_plain.unpack(q), s)
    return q.view(CODES[kind]).double() * s.double()[..., None]


def attention(query, kc, vc, ks, vs, kind, table, lens, scale, window=0):
    """(out, lse, out_bound, lse_bound) in 64 bits; NaN bounds nothing.

    The bounds, with u = 2^-24 for a rounding of fp32 and steps of 2u for a sum of the matrix units: a
    logit is a sum of D products (error at most 2 D u of the sum of their magnitudes) times two scales (4 u
    of it); 2^(s - m) takes the difference's rounding and its own (4 u (|s| + |m|) + 4 u); a weight times
    its vector's scale enters the products to 2^-18 of itself (2^-26 where queries are fp32, as queries
    then do); sums over n positions 2 n u.  Numerator and denominator both have the weights' error."""
    B, Hq, D = query.shape
    H, dv = kc.shape[2], vc.shape[3] * (2 if kind == "mxfp4" else 1)
    G, page_size, u = Hq // H, kc.shape[1], 2.0 ** -24
    out = torch.zeros(B, Hq, dv, dtype=torch.float64)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64)
    out_bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    entry = 2.0 ** -26 if query.dtype == torch.float32 else 2.0 ** -18
    for b in range(B):
        n = int(lens[b])
        first = max(0, n - window) if window else 0
        if n <= 0:
            continue
        if n > table.shape[1] * page_size:
            out[b], lse[b] = math.nan, math.nan
            continue
        p = torch.arange(first, n)
        pages = table[b].long()[p // page_size]
        if bool(((pages < 0) | (pages >= kc.shape[0])).any()):
            out[b], lse[b] = math.nan, math.nan
            continue
        k = vectors(kc, ks, kind, pages, p % page_size).permute(1, 2, 0)   # [H, D, n]
        v = vectors(vc, vs, kind, pages, p % page_size).permute(1, 0, 2)   # [H, n, dv]
        q = query[b].double().unflatten(0, (H, G))
        s = q @ k * scale
        size = q.abs() @ k.abs() * abs(scale)
        m = s.amax(-1, keepdim=True)
        w = torch.exp(s - m)
        total = w.sum(-1, keepdim=True)
        w = w / total
        o, reach = w @ v, w @ v.abs()
        logit = (2 * D + 4) * u * size
        off = (logit + 4 * u * (s.abs() + m.abs())).amax(-1, keepdim=True) + (4 + 2 * (n - first)) * u
        off = torch.expm1(off)
        out[b], out_bound[b] = o.flatten(0, 1), (reach * (2 * off + entry + 8 * u)).flatten(0, 1)
        lse[b] = (m + total.log()).flatten()
        lse_bound[b] = (off[..., 0] + 4 * u * (m[..., 0].abs() + total[..., 0].log() + 1)).flatten()
    return out, lse, out_bound, lse_bound


def near(got, want, bound, what):
    """got within bound of want, and a rounding to its own type; NaN and infinities where want has them."""
    got_type, got = got.dtype, got.detach().cpu().double()
    # past the type's largest value (and half a step) the nearest value of the type is an infinity
    past = want.abs() > torch.finfo(got_type).max * (1 + torch.finfo(got_type).eps / 4)
    want = torch.where(past & torch.isinf(got), torch.copysign(torch.full_like(want, math.inf), want),
                       want)
    plain = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN elsewhere"
    whole = ~plain & ~torch.isnan(want)
    assert torch.equal(got[whole], want[whole]), f"{what}: infinities differ"
    info = torch.finfo(got_type)
    # half a step of the type, of the value and of its bound; the smallest step below normal numbers
    room = bound + info.eps / 2 * (want.abs() + bound) + info.tiny * info.eps
    over = ((got - want).abs() - room)[plain]
    worst = ((got - want).abs() / room.clamp_min(1e-300))[plain]
    print(f"  {what}: at most {float(worst.max()) if worst.numel() else 0:.3f} of the bound", flush=True)
    assert not worst.numel() or float(over.max()) <= 0, f"{what}: {float(worst.max()):.3f} of the bound"


class PagePool:
    """The page pool as lists, one request after the other."""

    def __init__(self, table, lens, counts, page):
        self.table, self.lens, self.counts = table.tolist(), lens.tolist(), counts.tolist()
        self.page, self.columns = page, table.shape[1]

    def _fits(self, n):
        return 0 <= n <= self.columns * self.page

    def _held(self, n):
        return -(-n // self.page)

    def fork(self, parents, children):
        src, dst = [], []
        free = [p for p, c in enumerate(self.counts) if c <= 0]
        ended = False  # a fork that needs a page did not get one
        rows, lens = [list(r) for r in self.table], list(self.lens)
        for parent, child in zip(parents, children):
            ok = 0 <= parent < len(rows) and 0 <= child < len(rows) and self._fits(lens[parent])
            src.append(-1), dst.append(-1)
            if not ok:
                continue
            full, part = divmod(lens[parent], self.page)
            self.table[child], self.lens[child] = [-1] * self.columns, 0
            if part and (ended or not free):
                ended = True
                continue
            for c in range(full):
                page = self.table[child][c] = rows[parent][c]
                if 0 <= page < len(self.counts):
                    self.counts[page] += 1
            if part:
                src[-1], dst[-1] = rows[parent][full], free.pop(0)
                self.table[child][full], self.counts[dst[-1]] = dst[-1], 1
            self.lens[child] = lens[parent]
        return src, dst

    def extend(self, sequences, cu, num_tokens):
        slots, starts = [-1] * num_tokens, []
        free = [p for p, c in enumerate(self.counts) if c <= 0]
        ended = False
        for i, s in enumerate(sequences):
            add = cu[i + 1] - cu[i]
            starts.append(-1)
            if not 0 <= s < len(self.table) or add < 0 or not self._fits(self.lens[s]) or not self._fits(
                    self.lens[s] + add):
                continue
            old, have = self.lens[s], self._held(self.lens[s])
            need = self._held(old + add) - have
            if need and (ended or need > len(free)):
                ended = True
                continue
            for k in range(need):
                self.table[s][have + k] = free.pop(0)
                self.counts[self.table[s][have + k]] = 1
            self.lens[s], starts[-1] = old + add, old
            for t in range(add):
                column, offset = divmod(old + t, self.page)
                page = self.table[s][column]
                if 0 <= cu[i] + t < num_tokens and 0 <= page < len(self.counts):
                    slots[cu[i] + t] = page * self.page + offset
        return slots, starts

    def free(self, sequences):
        for s in sequences:
            if not 0 <= s < len(self.table) or not 0 < self.lens[s] <= self.columns * self.page:
                continue
            for page in self.table[s][:self._held(self.lens[s])]:
                if 0 <= page < len(self.counts):
                    self.counts[page] -= 1
            self.table[s], self.lens[s] = [-1] * self.columns, 0

    def compact(self):
        counts, src, dst = self.counts, [], []
        used = sum(c > 0 for c in counts)
        holes = [p for p in range(used) if counts[p] <= 0]
        for hole, page in zip(holes, [p for p in reversed(range(used, len(counts))) if counts[p] > 0]):
            src.append(page), dst.append(hole)
            counts[hole], counts[page] = counts[page], 0
        place = dict(zip(src, dst))
        self.table = [[place.get(p, p) for p in row] for row in self.table]
        behind = [-1] * (len(counts) // 2 - len(src))
        return src + behind, dst + behind, [used]
