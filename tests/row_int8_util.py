"""Reference of the row-scaled int8 products on the host: whole numbers in 64 bits, scales in the float32 steps that the kernels take."""
import torch

# Sizes of the GPU tests: odd numbers of rows and columns, rows that end inside a block of 128, one value of everything.
SHAPES = [(1, 1, 16), (1, 16, 16), (1, 40, 128), (2, 130, 272), (3, 4096, 512), (4, 129, 4096), (5, 64, 2112), (16, 300, 1024), (11, 530, 1040),
          (7, 4100, 512), (13, 257, 4096), (9, 40, 16), (16, 17, 4048), (17, 100, 640), (32, 256, 384), (33, 257, 1152), (64, 128, 4096),
          (65, 136, 1024), (100, 520, 528), (129, 384, 256), (200, 1000, 400), (257, 272, 1536), (520, 640, 2048), (1030, 528, 384)]
BACK_SHAPES = [(1, 1, 16), (1, 16, 16), (1, 130, 128), (5, 128, 272), (17, 300, 400), (64, 257, 640), (77, 1203, 1024), (130, 33, 2112), (200, 1000, 144),
               (300, 512, 512), (520, 264, 1040), (3, 9001, 144)]


def quantize(x):
    """Codes (int64) and scales (float32) of rows; a row with a NaN or an infinity has codes of zero and the scale NaN."""
    a = x.double().abs().amax(-1)
    bad = ~a.isfinite()
    a = a.masked_fill(bad, 1).clamp(min=2.0 ** -100)
    codes = torch.round(x.double().masked_fill(bad.unsqueeze(-1), 0) * 127 / a.unsqueeze(-1)).long()
    return codes, (a.float() / torch.tensor(127.0)).masked_fill(bad, float("nan"))


def sums(codes, w):
    """Whole sums, exact in float64 (below 2^53)."""
    return codes.double() @ w.double().t()


def product(x, w, scale, bias=None):
    """The product in x's dtype, by the kernels' own float32 steps: the whole sum, times the row's scale, times the column's, plus the bias, rounded once."""
    codes, xs = quantize(x)
    y = sums(codes, w).float() * xs.unsqueeze(-1) * scale
    return (y if bias is None else y + bias.float()).to(x.dtype)


def weight(gen, n, k, lead=(), std=0.02):
    codes, scale = quantize(torch.randn((*lead, n, k), generator=gen) * std)
    return codes.to(torch.int8), scale
