"""distill_loss and its gradient from their formulas in 64 bits, on the CPU, with the bounds that 32-bit arithmetic may be
off by.

An exponential's argument x (in units of 1 / T) is a difference and a product: off by 3 * 2^-24 |x| at most, and the
exponential itself by two steps, so e^x is off by (4 |x| + 4) 2^-24 of itself.  A sum of n positive numbers, in up to
`steps` additions in a row, is off by steps * 2^-24 of itself, and by its terms' own errors.  Rows of up to 1024 classes
add their weights p up as whole numbers of 2^-62, each cut to one: K entries are off by K 2^-62 at most, which counts
where p itself is smaller than 2^-38."""
import torch

EPS32 = 2.0 ** -24
INF = float('inf')


def reference(z, t, index, temperature, dloss=None, out_dtype=torch.float32):
    """z [rows, V], t and index [rows, K]: dict of each row's loss, whether it counts and, with dloss [rows], dz; and
    'tol_loss' and 'tol_dz' for 32-bit losses and gradients of out_dtype."""
    rows, v = z.shape
    z, t, index = z.detach().double().cpu() / temperature, t.detach().double().cpu() / temperature, index.cpu().long()
    counts = (index >= 0) & (index < v) & (t != -INF)
    live = counts.any(1)
    at = index.clamp(0, v - 1)
    t = torch.where(counts, t, torch.full_like(t, -INF))
    tm = torch.where(live, t.amax(1), torch.zeros(rows, dtype=torch.float64))[:, None]
    e = torch.exp(t - tm)
    s = torch.where(live, e.sum(1), torch.ones(rows, dtype=torch.float64))[:, None]
    p = e / s
    zm = z.amax(1, keepdim=True)
    ez = torch.exp(z - zm)
    zsum = ez.sum(1, keepdim=True)
    q = ez / zsum
    zi = (z - zm).gather(1, at)
    weighs = p > 0
    term = torch.where(weighs, p * ((t - tm) - zi), torch.zeros_like(p))
    ratio = torch.log(zsum / s)[:, 0]
    out = dict(loss=torch.where(live, temperature ** 2 * (term.sum(1) + ratio), torch.zeros_like(ratio)), live=live)
    steps = 64 + v / 256 + t.shape[1]

    def mean_size(w, x):  # of the arguments, by their weights
        return torch.where(w > 0, w * x.abs(), torch.zeros_like(w)).sum(1)
    size_t, size_z = mean_size(p, t - tm), mean_size(q, z - zm)
    size_of = torch.where(weighs, p * ((t - tm).abs() + zi.abs()) * (4 * (t - tm).abs() + 8), torch.zeros_like(p)).sum(1)
    whole = torch.where(weighs, p * ((t - tm).abs() + zi.abs()), torch.zeros_like(p)).sum(1)
    out['tol_loss'] = temperature ** 2 * EPS32 * (steps * (whole + 2 + ratio.abs()) + 4 * (size_t + size_z) + size_of
                                                  + 4 * size_t * whole) * live + 1e-36
    if dloss is not None:
        g = dloss.detach().double().cpu()[:, None] * temperature
        target = torch.zeros_like(q).scatter_add_(1, at, p)
        out['dz'] = torch.where(live[:, None], g * (q - target), torch.zeros_like(q))
        off_q = torch.where(q > 0, q * (steps + 8 + 4 * (z - zm).abs() + 4 * size_z[:, None]), torch.zeros_like(q))
        off_p = torch.where(weighs, p * (steps + 8 + 4 * (t - tm).abs() + 4 * size_t[:, None]), torch.zeros_like(p))
        off_p = torch.zeros_like(q).scatter_add_(1, at, off_p)
        info = torch.finfo(out_dtype)
        out['tol_dz'] = torch.where(live[:, None], EPS32 * g.abs() * (off_q + off_p) + t.shape[1] * 2.0 ** -62 * g.abs() + info.eps / 2 * out['dz'].abs()
                                    + info.tiny * info.eps + 1e-36 * g.abs(), torch.zeros_like(q))
    return out
