"""Plain implementations of the 4-bit cache (RDL_KV_Q4, include/rdl_attention.h):
blocks of 32 values, a head's page as one run of code bytes and scales."""
import torch

BLOCK, MOST = 32, 8160.0


def run_bytes(page, hd):
    return page * (hd // 2 + hd // BLOCK * 2)


def quantize(x):
    """(scales [..., hd / 32] f16, codes [..., hd] in 0 .. 15) of x [..., hd] f32, value by value in 64 bits."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    mag = b.abs().amax(-1)
    bits = (mag / 8).clamp(max=MOST).view(torch.int64)
    size = ((bits + (1 << 44) - 1 + (bits >> 45 & 1)) >> 45 << 45).view(torch.float64)  # 8 significant bits
    size = size.half().double()  # (only f16's smallest numbers have fewer)
    d = torch.where((b == mag[..., None]).any(-1), -size, size)
    code = torch.where(d[..., None] == 0, 0.0, torch.round(b / torch.where(d == 0, 1.0, d)[..., None]).clamp(-8, 7))
    d = torch.where(torch.isfinite(mag), d, float("nan"))
    return d.half(), (code.nan_to_num(0) + 8).to(torch.int64).flatten(-2)


def pack(codes):
    """Code bytes [..., hd / 2] of codes [..., hd]: words of 8, even codes in the low half's nibbles, odd ones in the high half's."""
    c = codes.unflatten(-1, (-1, 8))
    word = sum(c[..., e] << (4 * (e // 2) + 16 * (e % 2)) for e in range(8))
    return torch.stack([(word >> (8 * i) & 255).to(torch.uint8) for i in range(4)], -1).flatten(-2)


def unpack(b):
    """Codes [..., hd] of code bytes."""
    w = b.long().unflatten(-1, (-1, 4))
    word = w[..., 0] | w[..., 1] << 8 | w[..., 2] << 16 | w[..., 3] << 24
    return torch.stack([word >> (4 * (e // 2) + 16 * (e % 2)) & 15 for e in range(8)], -1).flatten(-2)


def values(scales, codes):
    """[..., hd] in 64 bits."""
    return ((codes - 8).double().unflatten(-1, (-1, BLOCK)) * scales.double()[..., None]).flatten(-2)


class Runs:
    """Views of a 4-bit pool's memory [pages, kv heads, run bytes (and more)]."""

    def __init__(self, mem, page, hd):
        self.page, self.hd = page, hd
        at = page * hd // 2
        self.codes = mem[..., :at].unflatten(-1, (page, hd // 2))
        self.scales = mem[..., at:run_bytes(page, hd)].view(torch.float16).unflatten(-1, (page, hd // BLOCK))

    def values(self):
        """[pages, kv heads, positions, hd] in 64 bits."""
        return values(self.scales, unpack(self.codes))

    def put(self, pages, offsets, x):
        """x [n, kv heads, hd] at offsets of pages."""
        d, c = quantize(x)
        self.scales[pages, :, offsets], self.codes[pages, :, offsets] = d, pack(c)
