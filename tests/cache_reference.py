"""Plain implementations of the paged-cache operators for the tests: rotary positions and attention
in 64 bits, the pages' bookkeeping in Python integers."""

from __future__ import annotations

import torch


def rotate(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, is_neox: bool) -> torch.Tensor:
    """x [T, heads, D] rotated, in float64."""
    y = x.double().clone()
    rot = table.shape[1]
    row = table[positions].double()
    cos, sin = row[:, None, : rot // 2], row[:, None, rot // 2 :]
    pairs = (slice(0, rot // 2), slice(rot // 2, rot)) if is_neox else (slice(0, rot, 2), slice(1, rot, 2))
    a, b = y[..., pairs[0]].clone(), y[..., pairs[1]].clone()
    y[..., pairs[0]] = a * cos - b * sin
    y[..., pairs[1]] = b * cos + a * sin
    return y


def rotary_bound(x: torch.Tensor, expected: torch.Tensor) -> torch.Tensor:
    """How far a rotated element may be from its value: half a bf16 unit in the last place (the
    unit is 2^-7 of the power of two below the value: at most 2^-8 of it) for the one rounding, and for
    three fp32 operations 2^-21 of the largest element of the head (each term is a product with a
    number of at most 1.5)."""
    return expected.abs() * 2.0**-8 + x.double().abs().amax(-1, keepdim=True) * 2.0**-21


def attention(q, key_cache, value_cache, tables, starts, lens, scale, window=0):
    """Output and its error scale sum(w |v|) / sum(w), float64 [T, heads, D]; rows of no sequence are NaN."""
    heads, kv_heads, page = q.shape[1], key_cache.shape[2], key_cache.shape[1]
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    size = out.clone()
    for s in range(len(lens)):
        begin, end, total = int(starts[s]), int(starts[s + 1]), int(lens[s])
        if end <= begin:
            continue
        position = torch.arange(end - begin, device=q.device) + (total - (end - begin))
        pages = tables[s, : -(-total // page)].long()
        k = key_cache[pages].double().flatten(0, 1)[:total]
        v = value_cache[pages].double().flatten(0, 1)[:total]
        key = torch.arange(total, device=q.device)
        seen = key[None, :] <= position[:, None]
        if window:
            seen &= key[None, :] > position[:, None] - window
        for h in range(heads):
            g = h // (heads // kv_heads)
            logits = (q[begin:end, h].double() @ k[:, g].T * scale).masked_fill(~seen, -torch.inf)
            top = logits.amax(-1, keepdim=True) if total else torch.full((end - begin, 1), -torch.inf, device=q.device).double()
            w = torch.where(seen, torch.exp(logits - top), 0.0)
            total_w = w.sum(-1, keepdim=True)
            inverse = torch.where(total_w > 0, 1.0 / total_w, 0.0)
            out[begin:end, h] = w @ v[:, g] * inverse
            size[begin:end, h] = w @ v[:, g].abs() * inverse
    return out, size


def attention_bound(expected: torch.Tensor, size: torch.Tensor) -> torch.Tensor:
    """Half a bf16 unit (at most 2^-8) of the result for its rounding and of each weight for the weights'; the
    scores of these inputs (at most 256 products, exact in fp32, of a total magnitude under 100 after
    scaling) are off by under 256 * 2^-24 * 100 * 2^-3 in practice, the exponentials by 2^-21, and
    fp32 sums by less: 2^-11 of the weights together."""
    return expected.abs() * 2.0**-8 + size * (2.0**-8 + 2.0**-11)


class Pool:
    """The pages' bookkeeping: tables as lists, counts, and data per page and token."""

    def __init__(self, tables, lens, refs, page_size):
        self.tables = [list(map(int, row)) for row in tables]
        self.lens = list(map(int, lens))
        self.refs = list(map(int, refs))
        self.page = page_size

    def pages(self, tokens):
        return -(-tokens // self.page)

    def _free(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def release(self, rows):
        for row in rows:
            for j, page in enumerate(self.tables[row]):
                if page >= 0:
                    self.refs[page] -= 1
                self.tables[row][j] = -1
            self.lens[row] = 0

    def reserve(self, rows, new_lens):
        """Number of pages lacking; nothing changes unless 0."""
        needs = [max(0, self.pages(n) - self.pages(self.lens[r])) for r, n in zip(rows, new_lens)]
        free = self._free()
        if sum(needs) > len(free):
            return sum(needs) - len(free)
        for row, new_len, need in zip(rows, new_lens, needs):
            have = self.pages(self.lens[row])
            for j in range(need):
                page = free.pop(0)
                self.tables[row][have + j] = page
                self.refs[page] = 1
            self.lens[row] = max(self.lens[row], new_len)
        return 0

    def fork(self, parents, children):
        """(pages lacking, [(source, target)]); nothing changes unless 0 are lacking."""
        lens = [self.lens[p] for p in parents]
        free = self._free()
        need = sum(n % self.page != 0 for n in lens)
        if need > len(free):
            return need - len(free), []
        copies = []
        for parent, child, n in zip(parents, children, lens):
            whole = n // self.page
            for j in range(whole):
                self.tables[child][j] = self.tables[parent][j]
                self.refs[self.tables[parent][j]] += 1
            if n % self.page:
                page = free.pop(0)
                self.tables[child][whole] = page
                self.refs[page] = 1
                copies.append((self.tables[parent][whole], page))
            self.lens[child] = n
        return 0, copies

    def compact(self):
        """(new tables, new counts, number in use, [(source, target)])."""
        live = sum(r > 0 for r in self.refs)
        holes = [i for i in range(live) if self.refs[i] <= 0]
        movers = [i for i in range(live, len(self.refs)) if self.refs[i] > 0]
        number = {i: i for i in range(len(self.refs))}
        number.update(zip(movers, holes))
        counts = [0] * len(self.refs)
        for i, r in enumerate(self.refs):
            if r > 0:
                counts[number[i]] = r
        tables = [[number.get(p, p) for p in row] for row in self.tables]
        return tables, counts, live, list(zip(movers, holes))
