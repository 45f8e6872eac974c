"""Plain forms of the 4-bit cache for its tests: encoding in float32 (which defines the stored bits) and the
values of records in float64, from the format's definition, column by column."""
import torch


def place(d, D, value):
    """(byte, shift) of column d's code in a record."""
    group, rest = divmod(d, 32)
    width = 4 if value else 8                     # columns of a word
    piece, first = divmod(rest, width)
    nibble = (piece * (D // 32) + group) * width + first
    return nibble // 2, 4 * (nibble % 2)


def encode(x, value):
    """float32 [..., D] -> uint8 records [..., D / 2 + D / 8]."""
    D = x.shape[-1]
    rec = torch.zeros(*x.shape[:-1], D // 2 + D // 8, dtype=torch.uint8, device=x.device)
    meta = torch.zeros(*x.shape[:-1], D // 16, dtype=torch.bfloat16, device=x.device)
    fifteenth = torch.tensor(1 / 15, dtype=torch.float32, device=x.device)
    for g in range(D // 32):
        c = x[..., 32 * g:32 * g + 32]
        lo, hi = c.amin(-1), c.amax(-1)
        s = ((hi - lo) * fifteenth).bfloat16()
        z = (lo + 8 * s.float()).bfloat16()
        meta[..., g], meta[..., D // 32 + g] = s, z
        s, z = s.float()[..., None], z.float()[..., None]
        code = (torch.where(s > 0, ((c - z) * (1 / s)).round(), 0.0) + 8).clamp(0, 15)
        code = torch.nan_to_num(code, nan=0.0).to(torch.uint8)
        for e in range(32):
            byte, shift = place(32 * g + e, D, value)
            rec[..., byte] |= code[..., e] << shift
    rec[..., D // 2:] = meta.view(torch.uint8)
    return rec


def parts(rec, D, value):
    """Codes less 8 [..., D], scales and midpoints [..., D] of records, float64."""
    meta = rec[..., D // 2:].contiguous().view(torch.bfloat16).double()
    group = torch.arange(D, device=rec.device) // 32
    code = torch.stack([(rec[..., place(d, D, value)[0]] >> place(d, D, value)[1]) & 15 for d in range(D)], -1)
    return code.double() - 8, meta[..., group], meta[..., D // 32 + group]


def decode(rec, D, value):
    c, s, z = parts(rec, D, value)
    return z + s * c


def turn(x, cos, sin, pairs):
    """Rotation in x's own type, each product and sum rounded once: [T, H, D] by [T, rot / 2]."""
    h = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    y = x.clone()
    a, b = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if pairs else (slice(0, h), slice(h, 2 * h))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def rotary_table(positions, rot, base=10000.0):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, rot, 2).double() / rot)
    return torch.cat((angle.cos(), angle.sin()), 1).float().cuda()
