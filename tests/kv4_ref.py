"""Plain float64 forms of the 4-bit cache (tests only), on numpy arrays: what rows become, and the planes' layout."""
import numpy as np

KEY_NIBBLE = (0, 4, 1, 5, 2, 6, 3, 7)
VALUE_NIBBLE = (0, 4, 2, 6)


def scales(x):
    """f16 scales of float64 blocks [..., 32]."""
    first = np.abs(np.where(np.isfinite(x), x, 0)).argmax(-1)
    m = np.take_along_axis(np.where(np.isfinite(x), x, 0), first[..., None], -1)[..., 0]
    part, e = np.frexp(np.abs(m) / 8)
    d = np.ldexp(np.rint(part * 32), e - 5)  # five significant bits, to nearest, ties to even
    d = np.minimum(d, 7936.0).astype(np.float16)
    d = np.where(m > 0, -d, d)
    return np.where(np.isfinite(x).all(-1), d, np.float16("nan"))


def quantize(x):
    """Codes [..., dim] and scales [..., dim / 32] of rows [..., dim]."""
    b = np.asarray(x, np.float64).reshape(x.shape[:-1] + (-1, 32))
    d = scales(b)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.clip(np.rint(b / d.astype(np.float64)[..., None]), -8, 7) + 8
    codes = np.where((d == 0)[..., None] | np.isnan(d)[..., None], 8, q).astype(np.uint8)
    return codes.reshape(x.shape), d


def values(codes, d):
    return ((codes.reshape(codes.shape[:-1] + (-1, 32)).astype(np.float64) - 8) * d.astype(np.float64)[..., None]).reshape(codes.shape)


def pack(codes, d, value):
    """The plane (bytes) of codes [pages, heads, page, dim] and scales [pages, heads, page, dim / 32]: element by element."""
    pages, heads, page, dim = codes.shape
    blocks = dim // 32
    plane = np.zeros((pages, heads, page // 16, 9 * dim), np.uint8)
    for r in range(16):
        for e in range(dim):
            if value:
                nib, dword = VALUE_NIBBLE[r % 4] + e % 2, ((r // 4) * 16 + e % 32 // 2) * blocks + e // 32
            else:
                nib, dword = KEY_NIBBLE[e % 8], ((e % 32 // 8) * 16 + r) * blocks + e // 32
            plane[..., 4 * dword + nib // 2] |= codes[:, :, r::16, e] << (4 * (nib % 2))
        for b in range(blocks):
            at = 8 * dim + 2 * (((r // 4) * blocks + b) * 4 + r % 4)
            plane[..., at:at + 2] = np.ascontiguousarray(d[:, :, r::16, b].astype(np.float16)).view(np.uint8).reshape(pages, heads, page // 16, 2)
    return plane


HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative


def bound(dtype, dim, n, long, out, spread, reach, largest):
    """How far an fp32 computation over the cache's values may be from the float64 one (out, spread and reach as in paged_ref.attend;
    largest: the largest value there is). The output's rounding (half a step); the weights' rounding: to the output's type in a long request that sees
    many keys, else to f16 (half a step of it is 2^-11) for bf16 and to two f16 terms (2^-21) for f16; fp32 sums of dim products in each
    score (dim 2^-24 of their absolute sum, entering numerator and denominator through e) and of n weights (n 2^-24), 2^-20 for exp2
    and the divide. Small weights: a weight times its value's scale stands in f16 numbers of 2^-24 at least, the row's largest weight being 2^6 at
    least above the largest scale's next power of two, so it is off by up to 2^-25 of 2^6 / 2, times codes of up to 8: 2^-30 of the largest
    value a key, 2^-25 of a weight in a long request. (fp32 exponentials end at 2^-126, far below.)"""
    half = HALF[dtype]
    weights = (half if long else 2.0 ** -11 if dtype == "bf16" else 2.0 ** -21) + 2 * dim * 2.0 ** -24 * reach + 2 * n * 2.0 ** -24 + 2.0 ** -20
    floor = n * 2.0 ** -30 * largest + (n * 2.0 ** -25 * spread if long and dtype == "f16" else 0.0)
    return half * np.abs(out) + (1 + half) * (weights * spread + floor) + (2.0 ** -25 if dtype == "f16" else 1e-38)
