"""Reference of the block-scaled fp8 products in 64 bits on the host, and inputs whose products are exact in any order of summation."""
import torch

E4M3 = torch.float8_e4m3fn


def blocks(n):
    return (n + 127) // 128


def e4m3(q):
    """q rounded to the nearest e4m3 number, ties to even; |q| <= 448."""
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(q / step) * step


def spread(scale, n, k, high):
    return scale.double().repeat_interleave(high, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]


def quantize(x, high):
    """Codes as numbers and scales (float32) of blocks of `high` x 128 of x [.., N, K]; blocks with a NaN or an infinity are NaN."""
    x = x.double()
    n, k = x.shape[-2:]
    pad = torch.nn.functional.pad(x.abs(), (0, -k % 128, 0, -n % high))
    a = pad.unflatten(-1, (-1, 128)).amax(-1).unflatten(-2, (-1, high)).amax(-2).clamp(min=2.0 ** -100)
    codes = e4m3(x * 448 / spread(a, n, k, high))
    return codes, (a.float() / 448).float()


def dense(codes, scale, high=128):
    return codes.double() * spread(scale, codes.shape[-2], codes.shape[-1], high)


def activations(gen, m, k, dtype, spread_bits=1):
    """Rows that quantize to themselves: whole numbers up to 8 and one 448 in each block, times a power of two."""
    x = torch.randint(-8, 9, (m, k), generator=gen).double()
    for b in range(0, k, 128):
        x[torch.arange(m), b + torch.randint(0, min(128, k - b), (m,), generator=gen)] = 448
        x[:, b:b + 128] *= torch.exp2(torch.randint(-spread_bits, spread_bits + 1, (m, 1), generator=gen).double())
    return x.to(dtype)


def weight(gen, n, k, base=0, lead=()):
    """Codes of whole numbers up to 8 and scales 2^(base - 1 .. base + 1).  A row's products with `activations` are multiples of
    2^(base - 2) below 2^(14 + base + 2) per block: sums over up to 32 blocks are exact in float32, and no product lies 13 bits below a
    neighbour (3584 against 1)."""
    codes = torch.randint(-8, 9, (*lead, n, k), generator=gen).float().to(E4M3)
    scale = torch.exp2(torch.randint(base - 1, base + 2, (*lead, blocks(n), blocks(k)), generator=gen).float())
    return codes, scale


def random_weight(gen, n, k, lead=(), std=0.02):
    codes, scale = quantize(torch.randn((*lead, n, k), generator=gen) * std, 128)
    return codes.float().to(E4M3), scale
