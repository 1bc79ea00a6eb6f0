"""Sizes of the 16-bit products that together reach every kernel, tile and split of them: (n, n_exp, R, K). The rules' test says so."""
DENSE = [(1, 72, 72), (1, 1032, 7176), (70, 4104, 7176), (520, 72, 7176), (520, 4104, 72), (900, 1032, 72), (1400, 1032, 7176), (2100, 72, 4104), (2100, 2056, 72),
         (2100, 4104, 72), (8500, 264, 7176)]
EXPERTS = [(1, 5, 72, 72), (1, 256, 72, 264), (40, 256, 72, 264), (300, 5, 1032, 72), (900, 256, 72, 2056), (1400, 5, 72, 4104), (1400, 5, 7176, 520), (1400, 5, 520, 7176),
           (2100, 5, 7176, 72), (4200, 5, 72, 72), (4200, 5, 72, 4104), (4200, 40, 1032, 72), (8500, 40, 520, 72), (8500, 5, 1032, 2056)]


def counts(n, ne):
    """slots of each expert, n together: the last has many, one in seven none, the others all sorts of tails"""
    if n < ne:
        return [int(e * n // ne != (e + 1) * n // ne) for e in range(ne)]
    c = [0 if e % 7 == 3 else min(n // ne * 2, 1 + 61 * e * e % max(2, n * 3 // (2 * ne))) for e in range(ne - 1)]
    while sum(c) > n:
        c[c.index(max(c))] //= 2
    return c + [n - sum(c)]
