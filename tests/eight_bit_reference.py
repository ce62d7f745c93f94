"""The operators on blocks of 8-bit numbers in 64 bits on the CPU, from their definition."""
import torch

BLOCK, LEAST = 128, -110


def blocks_of(x):
    """x [..., n] -> (numbers that the blocks stand for, exponents [..., blocks]), float64.  From the definition, by doubling."""
    x = x.detach().cpu().double()
    n = x.shape[-1]
    rows = x.reshape(-1, n)
    out, exps = torch.empty_like(rows), []
    for at in range(0, n, BLOCK):
        t = rows[:, at:at + BLOCK]
        finite = torch.isfinite(t)
        top = torch.where(finite, t.abs(), torch.zeros_like(t)).amax(1, keepdim=True)
        e = torch.full_like(top, float(LEAST))
        for _ in range(400):
            over = top * torch.exp2(-e) > 448
            if not over.any():
                break
            e += over.double()
        v = t * torch.exp2(-e)
        # the step of e4m3 at v: 2^-9 below 2^-5, twice as much from each power of two on
        step = torch.full_like(v, 2.0 ** -9)
        for k in range(-5, 9):
            step = torch.where(v.abs() >= 2.0 ** k, torch.full_like(v, 2.0 ** (k - 3)), step)
        r = torch.round(torch.where(finite, v, torch.zeros_like(v)) / step) * step
        r = torch.where((e == 120) & (r.abs() > 240), torch.sign(r) * 240, r)         # 256 2^120 is no fp32 number
        out[:, at:at + BLOCK] = torch.where(finite, r * torch.exp2(e), torch.full_like(v, float("nan")))
        exps.append(e)
    return out.reshape(x.shape), torch.cat(exps, 1).reshape(*x.shape[:-1], -1)


def q(x):
    return blocks_of(x)[0]


def phi(x):
    return torch.special.ndtr(x)


def gelu(x):
    return x * phi(x)


def gelu_slope(c):
    return phi(c) + c * torch.exp(-c * c / 2) * 0.3989422804014327


def layer_norm(x, weight, bias, eps, grad=None):
    """-> y, and with `grad` (dx, dweight, dbias), all of rows [R, n]; float64."""
    x64, w = x.detach().cpu().double(), weight.detach().cpu().double()
    mean = x64.mean(1, keepdim=True).float()
    kept = q(x.detach().cpu().float() - mean)
    c = x64 - mean.double()
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    y = c * r * w + bias.detach().cpu().double()
    if grad is None:
        return y
    dy = grad.detach().cpu().double()
    h, g = kept * r, dy * w
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return y, (dx, (dy * h).sum(0), dy.sum(0))
