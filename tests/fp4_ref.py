"""Plain NumPy forms of the 4-bit operators, in 64 bits with the roundings to float32 that the
definitions state, for the tests (test side only)."""
import numpy as np

E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
MID = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0])
E4M3_NORMALS = np.array([(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1])


def f32(v):
    return np.asarray(v, np.float64).astype(np.float32).astype(np.float64)


def quantize(x, fmt):
    """x (M, K) -> (E2M1 nibbles (M, K) u8, scale bytes (M, K/block) u8, row scales (M,))."""
    x = np.asarray(x, np.float64)
    M, K = x.shape
    block = 16 if fmt == "nvfp4" else 32
    b = x.reshape(M, K // block, block)
    if fmt == "nvfp4":
        amax = np.abs(x).max(axis=1)
        s = np.where(amax == 0, 1.0, np.maximum(f32(amax / 2688.0), 2.0 ** -120))
        inv = f32(1.0 / s)[:, None]
        top = f32(np.abs(b).max(axis=2) * inv)
        idx = np.minimum(np.searchsorted(6 * E4M3_NORMALS, top), len(E4M3_NORMALS) - 1)
        B = np.where(top == 0, 1.0, E4M3_NORMALS[idx])
        # byte: 8 codes per binade, the first normal is 0x08
        byte = np.where(top == 0, 0x38, idx + 8).astype(np.uint8)
        mul = f32(inv / B)
    else:
        s = np.ones(M)
        top = np.abs(b).max(axis=2)
        book = 2.0 ** np.arange(-40, 41)
        idx = np.minimum(np.searchsorted(6 * book, top), 80)
        e = np.where(top == 0, 0, idx - 40)
        B = 2.0 ** e
        byte = (e + 127).astype(np.uint8)
        mul = 1.0 / B
    y = f32(np.abs(b) * mul[..., None])
    code = np.searchsorted(MID, y.reshape(-1)).reshape(b.shape)  # a tie to the lower magnitude
    code = (code | np.where((b < 0) & (code != 0), 8, 0)).astype(np.uint8).reshape(M, K)
    return code, byte, s


def pack(nibbles):
    return (nibbles[:, 0::2] | (nibbles[:, 1::2] << 4)).astype(np.uint8)


def scale_values(byte, fmt):
    byte = byte.astype(np.int64)
    if fmt == "mxfp4":
        return 2.0 ** (byte.astype(np.float64) - 127)
    e, m = (byte >> 3) & 15, byte & 7
    return np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))


def values(nibbles, byte, fmt):
    """(rows, K) code * block scale, exact."""
    v = E2M1[nibbles & 7] * np.where(nibbles & 8, -1.0, 1.0)
    M, K = v.shape
    return (v.reshape(M, byte.shape[1], -1) * scale_values(byte, fmt)[..., None]).reshape(M, K)


def tile(byte):
    """Natural scale bytes (rows, S) -> scale tiles (flat), padding rows zero."""
    rows, S = byte.shape
    rb, words = -(-rows // 128), -(-S // 4)
    full = np.zeros((rb * 128, words * 4), np.uint8)
    full[:rows, :S] = byte
    return full.reshape(rb, 4, 32, words, 4).transpose(0, 3, 2, 1, 4).reshape(-1)


def tile_rows(rows, S):
    """Mask of the tile bytes that belong to rows < rows (padding rows are left unwritten)."""
    rb, words = -(-rows // 128), -(-S // 4)
    r = np.zeros((rb * 128, words * 4), bool)
    r[:rows] = True
    return r.reshape(rb, 4, 32, words, 4).transpose(0, 3, 2, 1, 4).reshape(-1)
