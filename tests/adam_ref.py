"""Oracle of the 8-bit moments in integer and fp32 steps on the CPU, from their definition."""
import numpy as np

M64 = (1 << 64) - 1


def mix(x):
    x = np.asarray(x, dtype=np.uint64)
    with np.errstate(over="ignore"):
        x = x + np.uint64(0x9E3779B97F4A7C15)
        x = (x ^ (x >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        x = (x ^ (x >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        return x ^ (x >> np.uint64(31))


def draws(n, seed, step, tensor):
    """(16 bits for m, 16 for v) of elements 0 .. n - 1."""
    key = mix(mix(seed) ^ np.uint64((step << 32) + tensor))
    i = np.arange(n, dtype=np.uint64)
    with np.errstate(over="ignore"):
        d = mix(key + (i >> np.uint64(1)))
    h = np.where(i & np.uint64(1), d >> np.uint64(32), d) & np.uint64(0xFFFFFFFF)
    return (h & np.uint64(0xFFFF)).astype(np.int64), (h >> np.uint64(16)).astype(np.int64)


def block_exps(x):
    """Exponent byte of each block of 256: the smallest e with max <= 1.875 2^(e - 127)."""
    out = []
    for b in range(0, len(x), 256):
        m = np.abs(x[b:b + 256].astype(np.float64)).max()
        if not np.isfinite(m):
            out.append(255)
            continue
        e = 1
        while m > 1.875 * 2.0 ** (e - 127) and e < 255:
            e += 1
        out.append(255 if e >= 254 else e)
    return np.array(out, dtype=np.uint8)


def values(codes, exps, top):
    """What codes stand for: sign 4 3 (top 15) or 5 3 (top 31)."""
    c = codes.astype(np.int64)
    mag = c & 127 if top == 15 else c
    field, man = mag >> 3, mag & 7
    v = np.where(field == 0, man / 8.0 * 2.0 ** (1 - top), (1 + man / 8.0) * 2.0 ** (field - top))
    e = np.repeat(exps.astype(np.int64), 256)[:len(c)]
    v = v * 2.0 ** (np.minimum(e, 254) - 127.0)
    if top == 15:
        v = np.where(c >= 128, -v, v)
    return np.where(e == 255, np.nan, v)


def codes_of(x, exps, top, draw):
    """Codes of fp32 x under block exponents: the float of x / scale, moved into the code's exponent
    range (subnormal codes are fp32 subnormals there), plus the draw in 20 bits, cut."""
    e = np.repeat(exps.astype(np.int64), 256)[:len(x)]
    y = np.abs(x).astype(np.float64) * 2.0 ** (127.0 - np.minimum(e, 253))
    y = (y * 2.0 ** (top - 127.0)).astype(np.float32)     # one rounding, of subnormals
    c = (y.view(np.uint32).astype(np.int64) + (draw << 4)) >> 20
    c = np.where(x > 0, np.maximum(c, 1), c) if top == 31 else c + 128 * (x < 0)
    return np.where(e == 255, 0, c).astype(np.uint8)
