"""The definitions of dense_reference.py in torch's float64, on whatever device the tensors are: for matrices that numpy takes too
long for.  test_gpu_nn_turns.py checks the two against each other."""
import torch


def kept(rows, width, p, seed, step, device, first=0):
    """Truth values [rows, width]: what dropout keeps in rows first, first + 1, .. (Philox4x32 with 7 rounds)"""
    low = 0xFFFFFFFF
    quads = -(-width // 4)
    at = torch.arange(first * quads, (first + rows) * quads, device=device)
    c = [at & low, at >> 32, torch.full_like(at, step & low), torch.full_like(at, step >> 32 & low)]
    k = [seed & low, seed >> 32 & low]
    for _ in range(7):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57             # modulo 2^64
        c = [(b >> 32 & low) ^ c[1] ^ k[0], b & low, (a >> 32 & low) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return torch.stack(c, 1).view(rows, quads * 4)[:, :width] >= round(p * 2 ** 32)


def factors(rows, width, drop, device):
    """What dropout multiplies by; drop: None or (p, seed, step)"""
    if drop is None:
        return torch.ones((), dtype=torch.float64, device=device)
    return kept(rows, width, *drop, device).double() / (1 - drop[0])


def statistics(x, eps):
    mean = x.mean(1, keepdim=True)
    return mean, 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()


def forward(x, weight, bias, eps):
    """y, mean, rstd of rows of float64 values, and what the rounding errors of each scale with"""
    mean, rstd = statistics(x, eps)
    h = (x - mean) * rstd
    y, near = h, x.abs() + mean.abs()
    off = (near + x.abs().mean(1, keepdim=True)) * rstd
    size = off + h.abs() * (1 + (off * h.abs()).mean(1, keepdim=True))      # the variance's own error moves every value of the row
    if weight is not None:
        y, size = y * weight, size * weight.abs()
    if bias is not None:
        y, size = y + bias, size + bias.abs()
    return (y, mean, rstd), (size, x.abs().mean(1, keepdim=True), rstd * (1 + (h.abs() * near * rstd).mean(1, keepdim=True)))


def gradient(dy, x, mean, rstd, weight):
    """(dx, dweight, dbias), and what the rounding errors of each scale with; mean and rstd: [rows, 1]"""
    h = (x - mean) * rstd
    g = dy if weight is None else dy * weight
    dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    off = h.abs() + (x.abs() + mean.abs()) * rstd
    size = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + off * (g * h).abs().mean(1, keepdim=True)
                   + h.abs() * (g.abs() * off).mean(1, keepdim=True))
    return (dx, (dy * h).sum(0), dy.sum(0)), (size, (dy.abs() * off).sum(0), dy.abs().sum(0))
