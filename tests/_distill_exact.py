"""distill_loss and its gradient in 50 decimal digits, for temperatures at which 64 bits lose theirs: of T^2 times a difference
of logarithms that agree in all but 1 / T^2 of themselves."""
from decimal import Decimal, localcontext


def reference(z, t, index, temperature):
    """z [rows, V], t and index [rows, K], every row with an entry that counts and logits that are finite or -infinity: each row's
    loss [rows], dz for dloss = 1 [rows, V], and the mean sizes of (z - max) / T and (t - max) / T [rows], as floats."""
    v = z.shape[1]
    losses, grads, sizes = [], [], []
    with localcontext() as ctx:
        ctx.prec = 50
        big_t = Decimal(temperature)
        for row, tr, ir in zip(z.detach().double().tolist(), t.detach().double().tolist(), index.tolist()):
            entries = [(Decimal(x) / big_t, i) for x, i in zip(tr, ir) if 0 <= i < v and x != -float('inf')]
            a = [Decimal(x) / big_t if x != -float('inf') else None for x in row]
            zm, tm = max(x for x in a if x is not None), max(x for x, _ in entries)
            ez = [Decimal(0) if x is None else (x - zm).exp() for x in a]
            es = [(x - tm).exp() for x, _ in entries]
            zsum, s = sum(ez), sum(es)
            ratio = (zsum / s).ln()
            loss = sum(e / s * ((x - tm) - (a[i] - zm)) for e, (x, i) in zip(es, entries)) + ratio
            dz = [e / zsum for e in ez]
            for e, (_, i) in zip(es, entries):
                dz[i] -= e / s
            losses.append(float(big_t * big_t * loss))
            grads.append([float(big_t * g) for g in dz])
            live = [x for x in a if x is not None]
            sizes.append(float(sum(zm - x for x in live) / len(live) + sum(tm - x for x, _ in entries) / len(entries)))
    return losses, grads, sizes
