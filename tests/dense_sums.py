"""Inputs on which the layers of any width are exact, and bounds of their sums over the samples that grow as the sums are taken.

Whole numbers: products of small whole numbers and their sums below 2^24 are whole numbers that 32 bits hold, so that no order of the sum and no
truncation changes them.  Every result is then one rounding of the exact value, and is compared bit by bit: a tile, a round or a part of a sum
that is left out or taken twice shows wherever its sum is not 0.

Random numbers: the weight gradient sums at most 512 samples in the tensor cores, each addition losing less than one unit of the last
place of a partial sum (2^-23 of it), adds these rounds up in 32 bits, and then at most one part for each of 148 SMs.  A column sum takes at
most n / 512 rows a thread ahead of 32 parts.  Both are off by at most (512 + n / 512 + 152) 2^-23 times the sum of the magnitudes."""
import torch


def whole(g, rows, width, t, most=2, step=1, pad=0, offset=0):
    """[rows][width] multiples of `step` up to most * step in magnitude, cut out of rows of width + pad entries `offset` entries behind a
    buffer's start."""
    full = torch.randint(-most, most + 1, (offset + rows * (width + pad),), device=g.device, generator=g).mul_(step).to(t)
    return full[offset:].view(rows, width + pad)[:, :width]


def sum_bound(n, magnitude):
    return (512 + n / 512 + 152) * 2.0 ** -23 * magnitude + 1e-40
