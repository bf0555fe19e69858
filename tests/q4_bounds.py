"""Entries whose groups differ in size, and how far an entry's values may be from what was stored."""
import torch


def inputs(device, rows, seed=0):
    """BF16 vectors [rows, 128]: entries of any size, each group 2^0 to 2^-18 of its entry; some beyond what is held, some all but nothing."""
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(rows, 4, 32, generator=g, device=device)
    x *= torch.exp2(-torch.randint(0, 19, (rows, 4, 1), generator=g, device=device).float())
    x *= torch.exp2(torch.randint(-66, 20, (rows, 1, 1), generator=g, device=device).float())
    return x.flatten(1).to(torch.bfloat16)


def bound(x):
    """With g the largest magnitude of a group and a that of its entry.  A scale lies within 1/32 of g / 7 of it, as long as it is one of 16 units or more: the
    value is off by half a step, g / 14 (1 + 1/32) (or, at the end of the codes, by g / 32).  Where 16 units are more than that, half a step is 8 units, and
    a unit is 2^-24 of a power of two that is a 2^9 / 7 at most: a / 28672, or 2^-61 where the power is the smallest.  Beyond the largest power a value is held as
    7 x 63488 x 2^-2 = 111104."""
    groups = x.double().clamp(-111104.0, 111104.0).unflatten(-1, (4, 32))
    g, a = groups.abs().amax(-1, keepdim=True), groups.abs().amax((-2, -1), keepdim=True)
    return torch.maximum(g / 14 * (1 + 2.0 ** -5), torch.maximum(a / 28672, torch.full_like(a, 2.0 ** -61))).expand_as(groups).flatten(-2) + (x.double().abs() - 111104.0).clamp(min=0)
