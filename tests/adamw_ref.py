"""numpy restatement of the AdamW step's 8-bit moments (csrc/d1_optim.hip): fp32 arithmetic in the
kernel's order, each operation rounded by itself, so codes are compared bit for bit."""
import numpy as np

BLOCK = 256


def mix(x):
    x = np.asarray(x, dtype=np.uint64)
    x = x ^ (x >> np.uint64(16))
    x = (x * np.uint64(0x9E3779B1)) & np.uint64(0xFFFFFFFF)
    x = x ^ (x >> np.uint64(15))
    x = (x * np.uint64(0xB7E15163)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def draws(seed, step, counters):
    c = np.asarray(counters, dtype=np.uint64)
    key = mix(mix(mix(seed & 0xFFFFFFFF) ^ np.uint64(seed >> 32)) ^ np.uint64(step))
    return mix((c & np.uint64(0xFFFFFFFF)) ^ mix(key ^ (c >> np.uint64(32))))


def blocks(x, n):
    out = np.zeros(-(-n // BLOCK) * BLOCK, x.dtype)
    out[:n] = x
    return out.reshape(-1, BLOCK)


def encode(x, top, draw16):
    """fp32 [n] -> (codes uint8 [n], exponents uint8 [blocks])."""
    n = len(x)
    a = blocks(np.abs(x).astype(np.float32), n)
    e = ((a.max(1).view(np.uint32).astype(np.int64) + 0xFFFFF) >> 23).astype(np.int64)
    y = np.ldexp(a.astype(np.float64), (top - e)[:, None]).astype(np.float32)
    code = (y.view(np.uint32).astype(np.int64) + (blocks(draw16.astype(np.int64), n) << 4)) >> 20
    code = np.minimum(code, (top + 1) * 8 - 1)
    if top == 31:
        code = np.where((code == 0) & (a > 0), 1, code)
    code = code.reshape(-1)[:n]
    if top == 15:
        code = code | np.where(x < 0, 128, 0)
    return code.astype(np.uint8), e.astype(np.uint8)


def decode(code, e, top):
    n = len(code)
    c = blocks(code.astype(np.uint32), n)
    a = ((c & np.uint32((top + 1) * 8 - 1)) << np.uint32(20)).astype(np.uint32).view(np.float32)
    x = np.ldexp(a.astype(np.float64), (e.astype(np.int64) - top)[:, None]).astype(np.float32).reshape(-1)[:n]
    return np.where(code >= 128, -x, x) if top == 15 else x


def moments(m, v, g, coef, b1=0.9, b2=0.999):
    """The new fp32 moments, every operation rounded to fp32."""
    f = np.float32
    d = g.astype(f) * f(coef)
    return (m * f(b1) + d * f(1.0 - b1)).astype(f), (v * f(b2) + (d * d) * f(1.0 - b2)).astype(f)
