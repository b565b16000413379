"""Rows, adapters and gradients of single products, which show what the bf16 matrix cores get of their 32-bit factors.

A 32-bit value is three bf16 p0 + p1 + p2, each what its upper sixteen bits hold of what the ones before left, an f16
value two, w0 + w1; those sums are exact.  A bf16 keeps eight bits, so with 2^e <= |x| < 2^(e+1) what p0 leaves is under
2^(e-7), what p1 leaves of that under 2^(e-15), and w1 is under 2^-7 |w|.  All products of two parts are exact in 32 bits.
Added up but for p2 w1 they are off by less than 2^-22 |x w| for that one and by half a step, 2^-24 |x w| at most, for
each of the four sums; a bf16 weight has three products and two sums, and none left out.
"""
import numpy as np

import lora_ref as ref

F32, F64, H = np.float32, np.float64, 2.0 ** -24


def product(bf):
    """How far the parts' product may be from the exact one, relative."""
    return 2 * H if bf else 2.0 ** -22 + 4 * H


def values(rng, shape, bits):
    """Values of so many bits, all of them in use, over a few powers of two."""
    m = 1 + rng.integers(0, 1 << (bits - 1), shape) / 2.0 ** (bits - 1)
    return rng.choice([-1.0, 1.0], shape) * m * 2.0 ** rng.integers(-3, 4, shape)


def upper(v):
    return (v.astype(F32).view(np.uint32) & 0xffff0000).view(F32)


def split(v, parts):
    """The parts that the kernels multiply."""
    got, rest = [], v.astype(F32)
    for _ in range(parts):
        got.append(upper(rest))
        rest = rest - got[-1]
    assert not rest.any()
    return got


def parts_product(x, w, bf, without=()):
    """x w of float32 arrays as the matrix cores have it: sums of the parts' products in 32 bits."""
    p, q = split(x, 3), split(w, 1 if bf else 2)
    total = np.zeros(np.broadcast_shapes(x.shape, w.shape), F32)
    for j in range(len(q)):
        for i in range(3 if j == 0 else 2):
            if (i, j) not in without:
                total = total + p[i] * q[j]
    return total


class Singles:
    """Every row of x and dy has one value, at columns that go through all; every row of B has one rank."""

    def __init__(self, lengths, adapters, rmax, out, cols, bf):
        rng = np.random.default_rng([sum(lengths), rmax, out, cols])
        self.lengths, self.seq, self.n, self.rmax, self.out, self.cols, self.bf = lengths, sum(lengths), adapters, rmax, out, cols, bf
        self.adapter = np.arange(len(lengths)).astype(np.int32) % adapters
        self.start = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
        self.rank, self.scale = np.full(adapters, rmax, np.int32), values(rng, adapters, 24).astype(F32)
        self.of = ref.owners(self.seq, self.start, self.adapter, adapters)
        rows = np.arange(self.seq)
        self.at, self.to = rng.permutation(self.seq) % cols, rng.permutation(self.seq) % out
        self.x, self.dy = np.zeros((self.seq, cols), F32), np.zeros((self.seq, out), F32)
        self.xv, self.dv = (values(rng, self.seq, 24).astype(F32) for _ in range(2))
        self.x[rows, self.at], self.dy[rows, self.to] = self.xv, self.dv
        bits = 8 if bf else 11
        self.a16, self.a = ref.to16(values(rng, (adapters, rmax, cols), bits), bf)
        b = np.zeros((adapters, out, rmax))
        self.only = np.arange(out) % rmax
        b[:, np.arange(out), self.only] = values(rng, (adapters, out), bits)
        self.b16, self.b = ref.to16(b, bf)

    def down_factors(self):
        """u[s, j] is one product: its two factors."""
        return np.broadcast_to(self.xv[:, None], (self.seq, self.rmax)), self.a[self.of, :, self.at].astype(F32)

    def up_factors(self, u):
        """y[s, o] is one product, times the scale: the two and that."""
        return u[:, self.only], self.b[self.of][:, np.arange(self.out), self.only].astype(F32), self.scale[self.of][:, None]

    def back_factors(self):
        """du has one value a row, dx [s, c] that times A: du's two factors, the scale, and A's row."""
        j = self.only[self.to]
        return self.dv, self.b[self.of, self.to, j].astype(F32), self.scale[self.of], self.a[self.of, j]
