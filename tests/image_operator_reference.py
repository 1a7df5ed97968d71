"""The operators of image and video models in 64 bits, from their definitions, and the error bounds their kernels are held to.

Bounds count roundings: u = 2^-24 for each fp32 operation, half a step (finfo.eps / 2) for the result's type."""
import numpy as np
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half a step among the type's subnormal numbers, where rounding is no longer relative."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def rounded(error, want, dtype):
    """Bound for a value known to `error` and then rounded to dtype."""
    return error * (1 + half_step(dtype)) + half_step(dtype) * want.abs() + smallest(dtype)


# -- rotary positions -------------------------------------------------------------
def frequencies(pairs, theta, arrangement):
    total, left, out, axis = sum(pairs), list(pairs), [], 0
    for i in range(total):
        while not left[axis]:
            axis = (axis + 1) % len(pairs)
        power = (pairs[axis] - left[axis]) / pairs[axis] if arrangement == "own" else i / total
        out.append((theta ** -power, axis))
        left[axis] -= 1
        if arrangement == "interleaved":
            axis = (axis + 1) % len(pairs)
    return out


def rope(x, positions, pairs, theta, arrangement, q, kv, layout, inverse=False):
    """(result, bound before rounding) of x [B, T, H, HS] (float64)."""
    f = frequencies(pairs, theta, arrangement)
    axis = torch.tensor([a for _, a in f], device=x.device)
    step = torch.tensor([v for v, _ in f], dtype=torch.float64, device=x.device)
    angle = positions.double()[axis].permute(1, 2, 0) * step
    cos, sin = angle.cos().unsqueeze(2), angle.sin().unsqueeze(2) * (-1 if inverse else 1)
    n, heads = len(f), q + kv
    first = slice(0, 2 * n, 2) if layout == "interleaved" else slice(0, n)
    second = slice(1, 2 * n, 2) if layout == "interleaved" else slice(n, 2 * n)
    a, b = x[:, :, :heads, first], x[:, :, :heads, second]
    out, bound = x.clone(), torch.zeros_like(x)
    out[:, :, :heads, first] = a * cos - b * sin
    out[:, :, :heads, second] = a * sin + b * cos
    # cos and sin: the reduced angle (at most pi/4) to three roundings, the polynomial to two, the rest below a tenth of one;
    # position * 2^-62 turns from the spectrum's last kept bit; the two products and the sum: two roundings of |a| + |b|
    far = 2 * np.pi * 2.0 ** -62 * float(positions.abs().max()) if positions.numel() else 0.0
    # the reference's own angle: position times frequency rounded to 53 bits, at most pi of it matters but its error is absolute
    far += 4 * 2.0 ** -53 * float(angle.abs().max()) if angle.numel() else 0.0
    e = (8 * U + far) * (a.abs() + b.abs())
    bound[:, :, :heads, first] = e
    bound[:, :, :heads, second] = e
    return out, bound


# -- group norm -------------------------------------------------------------------
# A statistic or a sum is a tree of partial results: at most 512 roundings lie between an element and the result
# (rows of a thread, threads of a column, runs of a sample).
CHAIN = 512 * U
# sigmoid for 16-bit storage: exponential to |z| + 2 roundings, a quotient to 2; 2^-19 for |z| up to 16, beyond which the
# error is below a 16-bit half step of the result.  fp32 storage: 8 roundings.


def sigmoid_error(dtype):
    return 8 * U if dtype == torch.float32 else 2.0 ** -19


def per_channel(stat, C):
    """[N, G] -> [N, 1, C]"""
    return stat.repeat_interleave(C // stat.shape[1], dim=1).unsqueeze(1)


def statistics(x, groups, eps):
    """mean, rstd of x [N, S, C] (float64), and the bound of the mean."""
    N, S, C = x.shape
    g = x.view(N, S, groups, C // groups)
    mean = g.mean(dim=(1, 3))
    var = (g - mean[:, None, :, None]).square().mean(dim=(1, 3))
    return mean, (var + eps).rsqrt(), CHAIN * g.abs().amax(dim=(1, 3))


def group_norm(x, w, b, groups, eps, silu, dtype):
    """((y, bound), (mean, bound), (rstd, bound)), bounds before rounding."""
    C = x.shape[2]
    mean, rstd, mean_error = statistics(x, groups, eps)
    # the variance follows to CHAIN plus what the mean's error adds, (mean_error rstd)^2; its square root halves that
    rstd_error = rstd * (CHAIN + (mean_error * rstd) ** 2)
    m, r, dm, dr = (per_channel(v, C) for v in (mean, rstd, mean_error, rstd_error))
    u = (x - m) * r
    z = u * w + b
    dz = w.abs() * (r * dm + u.abs() * (dr / r + 4 * U)) + 2 * U * (z.abs() + b.abs())
    if not silu:
        return (z, dz), (mean, mean_error), (rstd, rstd_error)
    y = z * torch.sigmoid(z)
    return (y, 1.1 * dz + sigmoid_error(dtype) * y.abs()), (mean, mean_error), (rstd, rstd_error)


def group_norm_backward(dy, x, mean, rstd, w, b, silu, dtype):
    """((dx, bound), (dweight, bound), (dbias, bound)) for the given mean and rstd [N, G]."""
    N, S, C = x.shape
    G = mean.shape[1]
    m, r = per_channel(mean, C), per_channel(rstd, C)
    u = (x - m) * r
    dz, dz_error = dy, torch.zeros_like(dy)
    if silu:
        z = u * w + b
        s = torch.sigmoid(z)
        dz = dy * s * (1 + z * (1 - s))
        # the derivative's factors: sigmoid, z (1 - sigmoid) with z to 4 roundings of |u w| + |b|; the second derivative is below 1/2
        dz_error = dy.abs() * ((sigmoid_error(dtype) + 8 * U) * (1 + z.abs()) * s + 0.5 * 4 * U * ((u * w).abs() + b.abs()))
    u_error = 2 * U * (x.abs() + m.abs()) * r + U * u.abs()
    db, dw = dz.sum(dim=(0, 1)), (dz * u).sum(dim=(0, 1))
    db_error = CHAIN * dz.abs().sum(dim=(0, 1)) + dz_error.sum(dim=(0, 1))
    dw_error = CHAIN * (dz * u).abs().sum(dim=(0, 1)) + (dz_error * u.abs() + dz.abs() * u_error).sum(dim=(0, 1))

    def mean_of(v):
        return per_channel(v.view(N, S, G, C // G).mean(dim=(1, 3)), C)

    d, d_error = w * dz, w.abs() * dz_error
    m1, m2 = mean_of(d), mean_of(d * u)
    m1_error = CHAIN * mean_of(d.abs()) + mean_of(d_error)
    m2_error = CHAIN * mean_of((d * u).abs()) + mean_of(d_error * u.abs() + d.abs() * u_error)
    dx = r * (d - m1 - u * m2)
    dx_error = r * (d_error + m1_error + u.abs() * m2_error + u_error * m2.abs() + 4 * U * (d.abs() + m1.abs() + (u * m2).abs()))
    return (dx, dx_error), (dw, dw_error), (db, db_error)


# -- dropout ------------------------------------------------------------------------
def philox(counter, key):
    """Philox4x32-10 on Python integers: the published algorithm, one block."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep_mask(n, seed, call, p, first=0):
    """Which of n elements from element `first` on (a multiple of 8) are kept, in numpy (uint64)."""
    group = np.arange(first // 8, first // 8 + (n + 7) // 8, dtype=np.uint64)
    lo, mask = np.uint64(32), np.uint64(0xFFFFFFFF)

    def blocks(second):
        c = [group & mask, (group >> lo) | np.uint64(second << 31), np.full_like(group, call & 0xFFFFFFFF), np.full_like(group, (call >> 32) & 0xFFFFFFFF)]
        k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
        for _ in range(10):
            a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(b >> lo) ^ c[1] ^ np.uint64(k[0]), b & mask, (a >> lo) ^ c[3] ^ np.uint64(k[1]), a & mask]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        out = np.empty((group.size, 8), dtype=np.uint64)
        for w in range(4):
            out[:, 2 * w], out[:, 2 * w + 1] = c[w] & np.uint64(0xFFFF), c[w] >> np.uint64(16)
        return out.reshape(-1)[:n]

    return ((blocks(0) << np.uint64(16)) | blocks(1)) >= np.uint64(round(p * 2 ** 32))
