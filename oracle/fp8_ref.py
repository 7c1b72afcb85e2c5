"""CPU restatement, in float64, of the 8-bit linear layer's operators
(quantisation to e4m3 blocks, the residual addition with its norm, the block
scaled matrix product). Test infrastructure only.

e4m3 (OCP "fn"): 1 sign, 4 exponent bits (bias 7), 3 mantissa bits, no
infinities, largest value 448, subnormal step 2^-9.
"""
import numpy as np

BLOCK = 128
AMAX_FLOOR = 2.0 ** -100


def e4m3(x):
    """float64 -> the nearest e4m3 value (ties to even), as float64; values
    past 448 saturate."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore"):
        exp = np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6)))
        step = 2.0 ** (exp - 3)
        return np.clip(np.rint(x / step) * step, -448.0, 448.0)


def block_amax(x, block_rows):
    """Largest magnitudes of the block_rows x 128 blocks of (rows, dim)."""
    rows, dim = x.shape
    rb, kb = -(-rows // block_rows), -(-dim // BLOCK)
    p = np.zeros((rb * block_rows, kb * BLOCK))
    p[:rows, :dim] = np.abs(x)
    return p.reshape(rb, block_rows, kb, BLOCK).max(axis=(1, 3))


def expand(scale, block_rows, rows, dim):
    """Scales of blocks -> one per element."""
    return np.repeat(np.repeat(scale, block_rows, 0)[:rows], BLOCK, 1)[:, :dim]


def quantize(x, block_rows=1):
    """(e4m3 values, scales) in float64."""
    x = np.asarray(x, np.float64)
    s = np.maximum(block_amax(x, block_rows), AMAX_FLOOR) / 448.0
    return e4m3(x / expand(s, block_rows, *x.shape)), s


def add_norm(x, y, gate, norm, weight, bias, scale, shift, eps, round_sum):
    """(out, h): x, y (B, L, dim); gate, scale, shift (B, dim); `round_sum`
    rounds h to the stream's type."""
    h = x if y is None else x + (y if gate is None else y * gate[:, None])
    h = round_sum(h)
    m = h.mean(-1, keepdims=True) if norm == "layer" else 0.0
    n = (h - m) / np.sqrt(((h - m) ** 2).mean(-1, keepdims=True) + eps)
    n = n if weight is None else n * weight
    n = n if bias is None else n + bias
    n = n if scale is None else n * (1 + scale[:, None])
    return (n if shift is None else n + shift[:, None]), h


def gelu_tanh(x):
    return 0.5 * x * (1 + np.tanh(np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3)))


def linear(xd, xs, wd, ws, bias=None, gelu=False):
    """(y, sum of |products| behind each y before the activation)."""
    x = xd * expand(xs, 1, *xd.shape)
    w = wd * expand(ws, BLOCK, *wd.shape)
    y, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        y, mag = y + bias, mag + np.abs(bias)
    return (gelu_tanh(y) if gelu else y), mag
