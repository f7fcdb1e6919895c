"""The 4-bit format and the routing restated in 64 bits with torch on the CPU or the GPU, from their definitions."""

import torch


def quantize(w, group):
    """(codes int64, scales float64 (..., rows, groups), values float64) of (..., rows, cols)."""
    w = torch.nan_to_num(w.double(), nan=0.0, posinf=float("inf"), neginf=-float("inf")).clamp(-2.0 ** 126, 2.0 ** 126)
    codes, scales = torch.empty(w.shape, dtype=torch.int64, device=w.device), []
    for lo in range(0, w.shape[-1], group):
        part = w[..., lo:lo + group]
        largest = part.abs().amax(-1, keepdim=True)
        first = (part.abs() == largest).to(torch.uint8).argmax(-1, keepdim=True)
        m, e = torch.frexp(part.gather(-1, first) / -8)
        s = torch.ldexp(torch.round(m * 32) / 32, e)
        s = torch.where(largest < 2.0 ** -100, torch.zeros_like(s), s)
        codes[..., lo:lo + group] = torch.where(s == 0, torch.zeros_like(part), torch.round(part / torch.where(s == 0, torch.ones_like(s), s))).clamp(-8, 7).long()
        scales.append(s)
    scales = torch.cat(scales, -1)
    return codes, scales, codes.double() * scales.repeat_interleave(group, -1)[..., :w.shape[-1]]


def pack(codes, scales, group):
    """One matrix as the header states the layout: 32-bit words of codes (as int64) and the bf16 scales."""
    rows, cols = codes.shape
    tiles, wide, groups = (rows + 15) // 16, (cols + 63) // 64, (cols + group - 1) // group
    out, out_scales = torch.full((tiles * wide * 128,), 0x88888888, dtype=torch.int64), torch.zeros(tiles * (groups + 1) * 16, dtype=torch.float64)
    r, k = torch.meshgrid(torch.arange(rows), torch.arange(cols), indexing="ij")
    rr, kk = r % 16, k % 64
    t, j, pair, h = kk % 32 // 8, 2 * (kk // 32) + kk % 8 // 4, kk % 4 // 2, kk % 2
    lane, reg = 4 * (rr % 8) + t, 2 * pair + rr // 8
    word = ((r // 16) * wide + k // 64) * 128 + lane * 4 + j
    shift = 4 * reg + 16 * h
    # every (word, shift) is met once: flip the bits of code 0 into those of the code
    flips = ((8 ^ (codes.cpu() + 8)) << shift).flatten()
    out ^= torch.zeros_like(out).index_add_(0, word.flatten(), flips)  # distinct bits of a word add up
    r, u = torch.meshgrid(torch.arange(rows), torch.arange(groups), indexing="ij")
    out_scales[((r // 16) * (groups + 1) + u) * 16 + 2 * (r % 8) + r % 16 // 8] = scales.cpu()
    r = torch.arange(rows)
    out_scales[((r // 16) * (groups + 1) + groups) * 16 + 2 * (r % 8) + r % 16 // 8] = scales.cpu().abs().amax(1)
    return out, out_scales.to(torch.bfloat16)


def product(x, values, bias=None):
    """(y, bound of the sums' error per unit of 2^-23) in 64 bits."""
    y = x.double() @ values.transpose(-1, -2)
    return (y if bias is None else y + bias.double()), x.double().abs() @ values.abs().transpose(-1, -2)


def tolerance(magnitude, y, K, dtype):
    """What a product's result may be off: every product is exact; a group's sum takes at most 8 steps of 16 terms, in which a term
    may be cut off at 2^-23 of the sum so far (plus two for the alignment), each group and each of at most 16 warps adds one rounding, planes and
    bias four more; then one rounding to the result's type."""
    steps = 10 + (K + 31) // 32 + 16 + 4
    return steps * 2.0 ** -23 * magnitude + (torch.finfo(dtype).eps / 2 * y.abs() * (1 + 2.0 ** -10) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps)


def route(ids, experts):
    """(order, position, offsets) by looking at one expert after the other."""
    flat = ids.flatten().tolist()
    order = [i for e in range(experts) for i, v in enumerate(flat) if v == e]
    position = [-1] * len(flat)
    for p, i in enumerate(order):
        position[i] = p
    offsets = [sum(1 for v in flat if 0 <= v < e) for e in range(experts + 1)]
    return (torch.tensor(order + [-1] * (len(flat) - len(order)), dtype=torch.int32), torch.tensor(position, dtype=torch.int32).view(ids.shape),
            torch.tensor(offsets, dtype=torch.int32))
