"""float64 definitions (torch, CPU) of the per-head norm, the position rotation and the
gradients, with first-order error bounds for float32 arithmetic, for the tests."""

import torch

U = 2.0 ** -24  # half a float32 step, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def pairs(dim, rotary, interleaved):
    """Element indices of the rotated pairs (first, second)."""
    i = torch.arange(rotary // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)


def rotate(x, cos, sin, interleaved):
    """R x for x [T, H, D] and cos / sin [T, R/2], one pair after the other."""
    y = x.clone()
    a, b = pairs(x.shape[-1], 2 * cos.shape[-1], interleaved)
    c, s = cos[:, None], sin[:, None]
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def rotate_abs(x, cos, sin, interleaved):
    """The sum of the absolute products behind each element of ``rotate``."""
    y = x.abs()
    a, b = pairs(x.shape[-1], 2 * cos.shape[-1], interleaved)
    c, s = cos[:, None].abs(), sin[:, None].abs()
    y[..., a], y[..., b] = (x[..., a].abs() * c + x[..., b].abs() * s, x[..., b].abs() * c + x[..., a].abs() * s)
    return y


def norm_rope(x, w, cos, sin, eps, interleaved):
    """y and the size of the terms behind each of its elements."""
    hat = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return rotate(hat * w, cos, sin, interleaved), rotate_abs(hat * w, cos, sin, interleaved)


def norm_rope_backward(x, w, g, cos, sin, eps, interleaved):
    """dx, dw and the sizes of the terms behind them."""
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    hat = x * r
    back, size = rotate(g, cos, -sin, interleaved), rotate_abs(g, cos, -sin, interleaved)
    dw, dw_size = (back * hat).sum((0, 1)), (size * hat.abs()).sum((0, 1))
    u = back * w
    dx = r * (u - hat * (u * hat).mean(-1, keepdim=True))
    dx_size = r * (size * w.abs() + hat.abs() * (size * w.abs() * hat.abs()).mean(-1, keepdim=True))
    return dx, dw, dx_size, dw_size


def positions_of(lens):
    return torch.cat([torch.arange(n) for n in lens]) if lens else torch.zeros(0, dtype=torch.long)
