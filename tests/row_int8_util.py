"""Reference of the row-scaled int8 products on the host: whole numbers in 64 bits, scales in the float32 steps that the kernels take."""
import torch

# Sizes of the GPU tests: odd numbers of rows and columns, rows that end inside a block of 128, one value of everything.
SHAPES = [(1, 1, 16), (1, 16, 16), (1, 40, 128), (2, 130, 272), (3, 4096, 512), (4, 129, 4096), (5, 64, 2112), (16, 300, 1024), (11, 530, 1040),
          (7, 4100, 512), (13, 257, 4096), (9, 40, 16), (16, 17, 4048), (17, 100, 640), (32, 256, 384), (33, 257, 1152), (64, 128, 4096),
          (65, 136, 1024), (100, 520, 528), (129, 384, 256), (200, 1000, 400), (257, 272, 1536), (520, 640, 2048), (1030, 528, 384)]
BACK_SHAPES = [(1, 1, 16), (1, 16, 16), (1, 130, 128), (5, 128, 272), (17, 300, 400), (64, 257, 640), (77, 1203, 1024), (130, 33, 2112), (200, 1000, 144),
               (300, 512, 512), (520, 264, 1040), (3, 9001, 144)]
# .. and sizes of every form of tiles, of both streaming kernels by number of waves, alone and in parts (test_every_form_is_run), and of the gradient
TILES = [(301, 702, 1040), (935, 1070, 144), (644, 1546, 1184), (653, 454, 4672), (1925, 4007, 144), (2250, 1806, 128), (3255, 2439, 144),
         (3466, 3630, 144), (1347, 1459, 128), (66, 2005, 7952), (2884, 130, 6560), (5000, 2050, 272), (6000, 4100, 144), (40, 3000, 4992), (20, 20011, 400), (48, 11009, 1040),
         (1700, 3001, 544), (4761, 794, 544), (2660, 3090, 144), (5132, 2498, 272), (1103, 19, 2048), (36, 20, 15904),
         (58, 7282, 720), (50, 5860, 1088), (150, 13824, 528), (1000, 4000, 1040), (513, 4090, 2064), (300, 5000, 1040), (500, 1700, 3216), (130, 2600, 8208)]
STREAMED = [(1, 2003, 16400), (2, 200, 8208), (4, 77, 8512), (3, 1001, 14656), (6, 4099, 4096), (16, 4096, 4112), (17, 512, 4096), (32, 200, 8192), (29, 783, 272),
            (13, 3037, 144), (5, 2000, 1040), (25, 2001, 2064), (2, 6990, 8832), (4, 20000, 528), (5, 17, 1424),
            (17, 18, 2880), (1, 17, 3616), (5, 16, 8064), (8, 40, 11712), (18, 16, 11552)]
BACK_TILES = [(130, 17, 7824), (1432, 736, 16), (5733, 1288, 16), (66, 865, 6064), (4026, 16, 2096), (8202, 16, 1552), (33, 710, 3376), (558, 18, 7200), (135, 1885, 7312), (66000, 17, 16), (2050, 300, 5200), (8200, 130, 1040), (3000, 520, 2320)]


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
