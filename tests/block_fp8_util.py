"""Reference of the block-scaled fp8 products in 64 bits on the host, and inputs whose products are exact in any order of summation."""
import torch

E4M3 = torch.float8_e4m3fn

# Sizes of the GPU tests.  The larger ones are there for the kernels that only they reach: odd numbers of rows and columns, K and N that end
# inside a block, and sums in parts.
SHAPES = [(1, 16, 16), (1, 1, 128), (1, 40, 128), (2, 130, 272), (3, 4096, 512), (4, 129, 4096), (5, 64, 2112), (16, 300, 1024), (11, 530, 1040), (7, 4100, 512), (13, 257, 4096), (9, 40, 16),
          (13, 17, 4832), (17, 100, 640),
          (32, 256, 384), (33, 257, 1152), (64, 128, 4096), (65, 136, 1024), (100, 520, 528), (129, 384, 256), (200, 1000, 400),
          (257, 272, 1536), (520, 640, 2048), (1030, 528, 384)]
TILES = [(301, 702, 1040), (935, 1070, 144), (1075, 23, 2032), (644, 1546, 1184), (653, 454, 4672), (1925, 4007, 144), (6017, 275, 7200),
         (2250, 1806, 128), (1606, 1155, 5280), (3255, 2439, 144), (5480, 267, 6928), (3466, 3630, 144), (1806, 2250, 17984),
         (1347, 1459, 128), (66, 2005, 7952), (1297, 777, 400), (2884, 130, 6560), (2692, 135, 7840),
         (1350, 707, 1520), (69, 1348, 7696), (5, 2839, 32544)]
BACK_SHAPES = [(1, 16, 16), (1, 130, 128), (5, 128, 272), (17, 300, 400), (64, 257, 640), (77, 1200, 1024), (130, 33, 2112), (200, 1000, 144),
               (300, 512, 512), (520, 264, 1040)]
BACK_TILES = [(130, 17, 7824), (33, 710, 3376), (558, 18, 7200), (135, 3885, 7312), (66000, 17, 16)]
EXPERTS = [(1, 2, 8, 128, 128), (1, 1, 1, 16, 128), (1, 8, 8, 400, 256), (2, 2, 16, 256, 384), (3, 4, 4, 272, 128), (40, 2, 5, 512, 256),
           (130, 3, 4, 144, 384), (300, 2, 70, 256, 128), (17, 5, 3, 384, 256), (600, 1, 2, 640, 512)]
EXPERT_TILES = [(39, 2, 70, 784, 128), (148, 1, 70, 800, 128), (56, 3, 70, 1712, 128), (1008, 4, 8, 160, 128), (897, 2, 20, 800, 128),
                (476, 3, 20, 2112, 128), (3356, 1, 8, 3344, 128), (2079, 2, 70, 128, 256), (2131, 2, 3, 128, 128),
                (225, 3, 20, 2064, 128), (488, 2, 20, 4016, 128), (399, 4, 20, 128, 896), (300, 2, 4, 640, 2304), (3000, 1, 7, 272, 1152),
                (286, 2, 8, 2864, 128), (2461, 4, 70, 448, 256), (3676, 4, 70, 288, 128), (1700, 2, 600, 16, 128), (1700, 2, 512, 16, 128), (900, 4, 2100, 16, 128),
                (9000, 2, 1, 16, 128), (70000, 1, 2, 16, 128)]

# Rows of each number of waves of the kernel of few rows, and tokens of each of the experts' second launch
FEW_ROWS = [(1, 40, 8336), (3, 130, 11008), (2, 17, 8208), (4, 64, 14336), (1, 8200, 8448), (2, 33, 272), (4, 40, 2048), (3, 70, 4112)]
FEW_PAIRS = [(1, 2, 4, 4112, 128), (2, 2, 8, 4096, 256), (1, 3, 8, 7168, 384), (1, 2, 4, 4096, 256), (2, 2, 8, 2048, 128)]


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
