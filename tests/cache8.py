"""What a cache in 8 bits holds, by its definition, on the host (no test in here)."""
import numpy as np

MOST = {"i8": np.float32(127), "e4m3": np.float32(448)}
TINY = np.float32(2.0 ** -126)


def _e4m3():
    """the values of the 127 codes without sign: 4 bits of exponent (bias 7), 3 of mantissa; code 127 is NaN"""
    c = np.arange(127)
    e, m = c >> 3, c & 7
    return np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0)).astype(np.float32)


E4M3 = _e4m3()
MIDDLES = ((E4M3[1:].astype(np.float64) + E4M3[:-1]) / 2).astype(np.float32)   # exact


def encode(x, kind):
    """fp32 values in units of codes -> bytes, to nearest, ties to the even code"""
    x = np.clip(np.asarray(x, np.float32), -MOST[kind], MOST[kind])
    if kind == "i8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    a = np.abs(x)
    low = np.searchsorted(MIDDLES, a, side="left")     # number of middles below a
    code = np.where((low < len(MIDDLES)) & (a == MIDDLES[np.minimum(low, len(MIDDLES) - 1)]), low + (low & 1), low)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def decode(code, kind):
    if kind == "i8":
        return code.view(np.int8).astype(np.float32)
    value = np.append(E4M3, np.float32(np.nan))[code & 127]
    return np.where(code & 128, -value, value)


class HostCache:
    """Codes [n_pages * page][kv][d] and scales [n_pages * page / block][kv] of keys and values, written as fdx_kv8_append_f32 says."""

    def __init__(self, n_pages, page, kv, dk, dv, kind, block):
        self.page, self.kv, self.kind, self.block = page, kv, kind, block
        self.codes = [np.zeros((n_pages * page, kv, d), np.uint8) for d in (dk, dv)]
        self.scales = [np.zeros((n_pages * page // block, kv), np.float32) for _ in (dk, dv)]

    def append(self, row_of, first, x, which):
        """x [n][kv][d]: positions first .. first + n - 1 of a sequence whose position p is in row row_of(p)"""
        codes, scales, kind, block = self.codes[which], self.scales[which], self.kind, self.block
        pos, last = first, first + len(x)
        while pos < last:
            begin = pos // block * block
            stop = min(last, begin + block)
            new, old, row0 = x[pos - first:stop - first], pos - begin, row_of(begin)
            for h in range(self.kv):
                with np.errstate(all="ignore"):
                    most, before = np.abs(new[:, h]).max(), scales[row0 // block, h] if old else np.float32(0)
                    if not (np.isfinite(most) and np.isfinite(before)):
                        codes[row0:row0 + old, h] = 0
                        codes[row0 + old:row0 + stop - begin, h] = 0
                        scales[row0 // block, h] = np.nan
                        continue
                    s = max(np.float32(most / MOST[kind]), TINY, before)
                    if old and s != before:
                        codes[row0:row0 + old, h] = encode(decode(codes[row0:row0 + old, h], kind) * np.float32(before / s), kind)
                    codes[row0 + old:row0 + stop - begin, h] = encode(new[:, h] * np.float32(np.float32(1) / s), kind)
                    scales[row0 // block, h] = s
            pos = stop

    def values(self, rows, which):
        """in 64 bits, [len(rows)][kv * d]"""
        rows = np.asarray(rows, np.int64)
        x = decode(self.codes[which][rows], self.kind).astype(np.float64) * self.scales[which][rows // self.block][:, :, None].astype(np.float64)
        return x.reshape(len(rows), x.shape[1] * x.shape[2])
