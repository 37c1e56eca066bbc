"""Plain forms of the low-precision operators for the tests: norms and products in 64 bits, e4m3 blocks step by step
in 32 (their definition), on whatever device the inputs are."""
import torch

F8 = torch.float8_e4m3fn
TINY = 2.0 ** -96


def unit(dtype):
    """Largest relative error of a rounding to `dtype`: half a step."""
    return torch.finfo(dtype).eps / 2


def floor(dtype):
    """Half a step below the smallest normal number: what a rounding there may lose absolutely."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _factor(a):
    return torch.ones_like(a).div(a) * 448.0


def _share(a):
    return a * torch.tensor(1.0 / 448.0, dtype=torch.float32, device=a.device)


def quantise(x, block_rows=1):
    """codes, scales of x (rows, cols) in blocks of (block_rows, 128)."""
    x = x.float()
    rows, cols = x.shape
    kb, rb = (cols + 127) // 128, (rows + block_rows - 1) // block_rows
    pad = torch.zeros(rb * block_rows, kb * 128, device=x.device)
    pad[:rows, :cols] = x
    a = pad.view(rb, block_rows, kb, 128).abs().amax(3).amax(1)
    a = torch.maximum(a, torch.tensor(TINY, device=x.device))  # NaN stays NaN
    f = _factor(a).repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    return (x * f).to(F8), _share(a)


def values(codes, scales):
    """Codes and scales (one per row or per 128 rows) as 64-bit values."""
    rows, cols = codes.shape
    s = scales.double()
    if s.size(0) != rows:
        s = s.repeat_interleave(128, 0)[:rows]
    return codes.double() * s.repeat_interleave(128, 1)[:, :cols]


def same_codes(a, b):
    """Equal e4m3 values, NaN equal to NaN, zeros of either sign equal."""
    x, y = a.float(), b.float()
    return torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(torch.nan_to_num(x), torch.nan_to_num(y))


def moments_to_blocks(m, v):
    """32-bit moments -> codes of m, codes of sqrt(v), scales, the blocks of 256 of AdamW's 8-bit moments."""
    n = m.numel()
    out, scales = [], []
    for u, root in ((m, False), (v.sqrt(), True)):
        pad = torch.zeros((n + 255) // 256 * 256, device=m.device)
        pad[:n] = u.reshape(-1)
        pad = pad.view(-1, 256)
        a = torch.maximum(pad.abs().amax(1, keepdim=True), torch.tensor(TINY, device=m.device))
        c = pad * _factor(a)
        if root:
            c = torch.where(pad > 0, c.clamp_min(2.0 ** -9), c)
        out.append(c.to(F8).view(-1)[:n].view(m.shape))
        scales.append(_share(a))
    return out[0], out[1], torch.cat(scales, 1)


def moments_from_blocks(mc, rc, scales):
    n = mc.numel()
    out = []
    for c, s in ((mc, scales[:, :1]), (rc, scales[:, 1:])):
        pad = torch.zeros((n + 255) // 256 * 256, device=mc.device)
        pad[:n] = c.reshape(-1).float()
        out.append((pad.view(-1, 256) * s).view(-1)[:n].view(mc.shape))
    return out[0], out[1] * out[1]
