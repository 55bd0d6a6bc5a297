"""Products of which each runs a kernel form of its own, ends inside a tile on either side, and has blocks with scales of their own."""
import torch

# form, results in 16 bits or in 32, rows, n, k.  Of the tiles of 256 rows: even and odd numbers of blocks along k, fewer and more tiles than compute units.
CASES = [
    (0, 16, 13, 333, 1000), (0, 32, 7, 129, 700), (32, 16, 30, 333, 1000), (32, 32, 27, 300, 385), (64, 16, 61, 333, 1000), (64, 32, 50, 300, 385),
    (128, 16, 1001, 700, 300), (128, 32, 1001, 700, 300), (128, 16, 257, 641, 520), (128, 32, 257, 641, 520),
    (192, 16, 2695, 4353, 391), (192, 16, 7121, 1676, 265), (192, 16, 8702, 2819, 434), (192, 16, 7586, 3230, 778),
    (192, 32, 2695, 4353, 391), (192, 32, 7121, 1676, 265), (192, 32, 8702, 2819, 434), (192, 32, 8506, 2857, 513),
    (256, 16, 1814, 6579, 385), (256, 16, 7630, 1546, 262), (256, 16, 7871, 3658, 129), (256, 16, 8720, 3238, 772),
    (256, 32, 1814, 6579, 385), (256, 32, 1671, 7028, 513), (256, 32, 3660, 7821, 641), (256, 32, 5251, 5420, 513),
]


def blocks(rows, cols, block_rows, device, seed):
    """0 and +-1, each block of block_rows x 128 times a power of two of its own (1, 2, 4 or 8)."""
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randint(-1, 2, (rows, cols), generator=g, device=device).float()
    power = torch.randint(0, 4, (-(-rows // block_rows), -(-cols // 128)), generator=g, device=device).float().exp2()
    return x * power.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
