"""GPU: draws whose level lies on the border beside columns that weigh nothing.

A draw sums weights lane by lane in a fixed order, so the running sum of a lane behind a border may exceed the border by a last bit although the lane adds nothing.
Which columns can be drawn must not hang on that bit.  The rows here are made for it: the kernel's sums are repeated on the CPU bit for bit (IEEE double, libm's fma),
and a few logits are tuned until the level is the very border."""
import ctypes
import math
import struct

import numpy as np
import pytest
import torch

from tests import policy_reference as R

fma = ctypes.CDLL("libm.so.6").fma
fma.restype, fma.argtypes = ctypes.c_double, [ctypes.c_double] * 3

POLY = [float.fromhex(h) for h in ("0x1.b63880f05fbb6p-24", "0x1.63d136346743dp-20", "0x1.ffcb95155e91bp-17", "0x1.4308ac85ac496p-13", "0x1.5d87fe86fe9e5p-10",
                                   "0x1.3b2ab7181b749p-7", "0x1.c6b08d7047e52p-5", "0x1.ebfbdff823cedp-3", "0x1.62e42fefa39efp-1", "0x1p0")]
K2 = 1.4426950408889634074
SHIFT = 1.5 * 2.0 ** 52
C = 4   # float32 columns a lane


def weight(y):
    """The kernel's exp(y) at temperature 1; of -inf it is 2^-1000."""
    y = max(y, -1000.0 * 0.69314718055994530942)
    shifted = fma(y, K2, SHIFT)
    n = shifted - SHIFT
    f = fma(y, K2, -n)
    p = POLY[0]
    for c in POLY[1:]:
        p = fma(p, f, c)
    return math.ldexp(p, int(n))


def running_sums(v):
    """Of 64 lanes: shifts by 1, 2, 4, 8 inside rows of 16, then the rows' last lanes."""
    v = list(v)
    for s in (1, 2, 4, 8):
        v = [x + (v[i - s] if i % 16 >= s else 0.0) for i, x in enumerate(v)]
    v = [x + (v[i // 16 * 16 - 1] if i // 16 in (1, 3) else 0.0) for i, x in enumerate(v)]
    return [x + (v[31] if i >= 32 else 0.0) for i, x in enumerate(v)]


def total(v):
    """Of 64 lanes, by exchanges."""
    v = list(v)
    for other in (lambda i: i ^ 1, lambda i: i ^ 2, lambda i: i // 8 * 8 + 7 - i % 8, lambda i: i // 16 * 16 + 15 - i % 16, lambda i: i ^ 16, lambda i: i ^ 32):
        v = [x + v[other(i)] for i, x in enumerate(v)]
    return v[0]


def lane_sum(ys):
    s = 0.0
    for y in ys:
        s += weight(y)
    return s


def floats_below(lo, hi, good):
    """The greatest negative float32 in [lo, hi] that is `good`, which is monotone (true below some border): by its bits."""
    a, b = (struct.unpack("<I", struct.pack("<f", -v))[0] for v in (hi, lo))   # of negative floats: a greater pattern is a lesser value
    value = lambda bits: -struct.unpack("<f", struct.pack("<I", bits))[0]
    while a < b:
        mid = (a + b) // 2
        if good(value(mid)):
            b = mid
        else:
            a = mid + 1
    return value(a)


def tuned(sum_of, want):
    """Four negative logits for which sum_of(them) is `want`, coarse to fine, or None."""
    ys = [-math.inf] * C
    for j, (lo, hi) in enumerate(((-14.0, -1e-6), (-32.0, -13.0), (-50.0, -29.0))):
        def good(y):
            ys[j] = y
            return sum_of(ys) <= want
        ys[j] = floats_below(lo, hi, good)
        if not good(ys[j]):
            ys[j] = -math.inf
    return ys if sum_of(ys) == want else None


def border(parts, empty, add, u):
    """(logits to put into the last part, level) such that the level u * (whole sum) is exactly the running sum before part `empty`, which exceeds it; or None."""
    upto = running_sums(parts)
    low, high = upto[empty - 1], upto[empty]
    if not high > low:
        return None
    s = low / u
    for k in range(-4, 5):
        want = s + k * math.ulp(s)
        if low <= u * want < high:
            ys = tuned(add, want)
            if ys:
                return ys, u * want
    return None


def wave_row(rng, u):
    """256 logits, a vector of a wave's lane each: lane `empty` masked, the lanes behind it too but the last."""
    for _ in range(400):
        empty = int(rng.integers(3, 60))
        x = np.float32(-6 - 6 * rng.random((64, C)))
        open_ = np.zeros((64, C), bool)
        open_[:empty] = True
        open_[63] = True
        lanes = [lane_sum(x[i] if open_[i, 0] else [-math.inf] * C) for i in range(63)]
        found = border(lanes + [0.0], empty, lambda ys: total(lanes + [lane_sum(ys)]), u)
        if found:
            x[63], level = found[0], found[1]
            sums = lanes + [lane_sum(x[63])]
            assert u * total(sums) == level
            first = next(i for i, s in enumerate(running_sums(sums)) if s > level)
            assert first == empty   # the lane that the running sums alone point at: it weighs 64 x 2^-1000 of nothing
            return x.reshape(-1), open_.reshape(-1)
    raise AssertionError("no such row found")


def workgroup_row(rng, u):
    """4,096 logits, 16 parts of a wave's vectors each: part `empty` masked, those behind it too but the last."""
    for _ in range(40):
        empty = int(rng.choice([3, 5, 7, 9, 11, 13]))
        x = np.float32(-8 - 6 * rng.random((16, 64, C)))
        open_ = np.zeros((16, 64, C), bool)
        open_[:empty] = True
        open_[15, 63] = True
        none = [lane_sum([-math.inf] * C)] * 64
        parts = [total([lane_sum(v) for v in x[i]]) if open_[i, 0, 0] else total(none) for i in range(15)]
        last = lambda ys: total(none[:63] + [lane_sum(ys)])

        def whole(ys):   # each of the four waves adds up its vectors' sums, then the workgroup the waves'
            p = parts + [last(ys)]
            waves = [((0.0 + p[w] + p[4 + w]) + p[8 + w]) + p[12 + w] for w in range(4)]
            return ((waves[0] + waves[1]) + waves[2]) + waves[3]

        found = border(parts + [0.0] * 49, empty, whole, u)
        if found:
            x[15, 63], level = found[0], found[1]
            sums = parts + [last(x[15, 63])] + [0.0] * 48
            first = next(i for i, s in enumerate(running_sums(sums)) if s > level)
            assert first == empty and u * whole(x[15, 63]) == level
            return x.reshape(-1), open_.reshape(-1)
    raise AssertionError("no such row found")


ROWS, SEED = 4, 20


def rows_on_the_border(make):
    rng = np.random.default_rng(7)
    us = R.uniforms(64, SEED)
    keys = [k for k in range(64) if 0.3 < float(us[k]) < 0.8][:ROWS]
    made = [make(rng, float(us[k])) for k in keys]
    return torch.tensor(np.stack([m[0] for m in made])), torch.from_numpy(np.stack([m[1] for m in made])), torch.tensor(keys)


@pytest.mark.parametrize("make", [wave_row, workgroup_row])
def test_rows_on_the_border_can_be_made(make):
    x, allowed, keys = rows_on_the_border(make)
    assert x.shape == allowed.shape and len(keys) == ROWS and not allowed.all(1).any()


@pytest.mark.gpu
@pytest.mark.parametrize("make", [wave_row, workgroup_row])
def test_a_level_on_the_border_never_takes_a_column_that_weighs_nothing(make):
    from gym_amd.policy import LogitRules, pack_action_mask, sample_actions
    x, allowed, keys = rows_on_the_border(make)
    rules = LogitRules(mask=pack_action_mask(allowed.cuda()))
    s = sample_actions(x.cuda(), rules, seed=SEED, rows=keys.cuda())
    at = s.actions.cpu().long()
    assert allowed.gather(1, at[:, None]).all(), at
    assert torch.isfinite(s.log_prob).all()
    # the running sum passes the level with the next column that weighs anything
    for b in range(ROWS):
        tail = torch.nonzero(allowed[b])[:, 0]
        assert int(at[b]) == int(tail[tail >= x.shape[1] - C][0]) or int(at[b]) == int(tail[tail < x.shape[1] - C][-1]), b
