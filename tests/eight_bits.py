"""A paged cache in 8 bits from its definition: blocks of 16 positions of a
page and head, held as e4m3 values times the smallest power of two that brings
the largest of their rows to at most 448.

Elements come as 64-bit numbers that 32 bits hold. Multiplying by a power of two
and rounding to e4m3 once are both exact operations on them, so a kernel's
codes and scales have no tolerance.
"""
import torch

LOW, HIGH = -100, 119


def scale_of(top: float) -> float:
    """The scale of a block whose largest finite element is top."""
    e = LOW
    while e < HIGH and top > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def round8(x: torch.Tensor) -> torch.Tensor:
    """x (64 bits, finite) to the nearest of 0, +-2^-9 .. +-448, ties to even, and 448 past it."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -60))).clamp_min(-6.0) - 3.0)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def form(rows: torch.Tensor):
    """(values, scale) of a block's rows [n, dim] in 64 bits: what the codes are, NaN where an element is not finite."""
    fine = torch.isfinite(rows)
    scale = scale_of(float(rows[fine].abs().max()) if bool(fine.any()) else 0.0)
    return torch.where(fine, round8(torch.where(fine, rows, 0.0) / scale), float("nan")), scale


def turn(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x [rows, heads, dim] (fp32) turned by the angles of cos and sin [rows, half]: products and sums are each rounded to fp32."""
    half = cos.shape[1]
    x = x.clone()
    cos, sin = cos[:, None], sin[:, None]
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., one].clone(), x[..., two].clone()
    x[..., one], x[..., two] = a * cos - b * sin, b * cos + a * sin
    return x


class Copy:
    """A cache's tensors on the CPU, and what its steps do to them."""

    def __init__(self, cache):
        self.page, self.layers, self.heads = cache.page_size, cache.n_layers, cache.kv_heads
        self.wide = cache.scales is None
        self.pool = cache.pool.cpu() if self.wide else cache.pool.cpu().double()
        self.scales = None if self.wide else cache.scales.cpu().double()
        self.table, self.lengths = cache.page_table.cpu().clone(), cache.lengths.cpu().clone()

    def place(self, slot, position):
        return int(self.table[slot, position // self.page]), position % self.page

    def row(self, layer, which, head, slot, position):
        p, r = self.place(slot, position)
        x = self.pool[layer, which, p, head, r]
        return x if self.wide else x * self.scales[layer, which, p, head, r // 16]

    def put(self, layer, which, head, slot, first, rows):
        """Rows (64 bits) at positions first ..; blocks are formed from their rows below `first` and these."""
        if self.wide:
            for i, x in enumerate(rows):
                p, r = self.place(slot, first + i)
                self.pool[layer, which, p, head, r] = x.to(self.pool.dtype)
            return
        for start in range(first // 16 * 16, first + len(rows), 16):
            old = [self.row(layer, which, head, slot, j) for j in range(start, max(start, min(first, start + 16)))]
            new = [rows[j - first] for j in range(max(start, first), min(start + 16, first + len(rows)))]
            values, scale = form(torch.stack(old + new))
            p, r = self.place(slot, start)
            self.pool[layer, which, p, head, r:r + len(values)] = values
            self.scales[layer, which, p, head, r // 16] = scale

    def commit(self, slot, accepted):
        n, first = len(accepted), int(self.lengths[slot])
        for layer in range(self.layers):
            for which in range(2):
                for head in range(self.heads):
                    rows = [self.row(layer, which, head, slot, first + j).clone() for j in accepted]
                    for start in range(first // 16 * 16, first + n, 16):
                        here = range(max(0, start - first), min(n, start + 16 - first))
                        if all(accepted[i] == i for i in here):
                            continue  # no row moves: the block stays as it is
                        self.put(layer, which, head, slot, first + here[0], [rows[i] for i in here])
        self.lengths[slot] += n

    def same(self, cache):
        assert torch.equal(cache.lengths.cpu(), self.lengths)
        got = cache.pool.cpu() if self.wide else cache.pool.cpu().double()
        assert torch.equal(got.isnan(), self.pool.isnan())
        assert torch.equal(got.nan_to_num(0.0), self.pool.nan_to_num(0.0))
        if not self.wide:
            assert torch.equal(cache.scales.cpu().double(), self.scales)
