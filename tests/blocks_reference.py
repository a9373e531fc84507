"""What the ops of decoder layers in 8 and 4 bits compute, in numpy: quantization
operation for operation in 32 bits (so codes and scales can be compared bit for
bit), everything else from its definition in 64 bits."""
import numpy as np

F = np.float32


def half_step(dtype_name):
    """The largest rounding error of a type, relative to the value."""
    return {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype_name]


def smallest_step(dtype_name):
    """Half the distance of the smallest numbers of a type."""
    return {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}[dtype_name]


def e4m3(x):
    """The e4m3 codes nearest to f32 values within +-448, ties to even; NaN 0x7F."""
    x = np.asarray(x, F)
    v = np.abs(x).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        step = np.exp2(np.floor(np.log2(np.maximum(v, 2.0 ** -6))) - 3)
        q = np.rint(v / step) * step
    e = np.floor(np.log2(np.maximum(q, 2.0 ** -6)))
    code = np.where(q < 2.0 ** -6, q * 512, (e + 6) * 8 + q / np.exp2(e - 3))
    code = np.where(np.isnan(x), 127, code).astype(np.uint8)
    return np.where(np.signbit(x), code | 128, code).astype(np.uint8)


def quantize_blocks(x, rows):
    """(codes, scales) of f32 x [M, K]."""
    M, K = x.shape
    y = np.empty((M, K), np.uint8)
    s = np.empty((-(-M // rows), -(-K // 128)), F)
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            at = np.s_[i * rows:(i + 1) * rows, j * 128:(j + 1) * 128]
            b = x[at]
            top = F(np.fmax.reduce(np.abs(b), axis=None, initial=F(0)))
            s[i, j] = max(F(top / F(448)), F(2.0 ** -126))
            with np.errstate(invalid="ignore", over="ignore"):
                q = (b / s[i, j]).astype(F)
            y[at] = e4m3(np.where(q > 448, F(448), np.where(q < -448, F(-448), q)))
    return y, s


def spread(s, rows, M, K):
    """Scales as a [M, K] matrix in 64 bits."""
    return np.repeat(np.repeat(s.astype(np.float64), rows, 0)[:M], 128, 1)[:, :K]


def rotate(x, cos, sin, rot, interleaved):
    """x [B, H, S, D], cos and sin [B, S, rot / 2]; 64 bits."""
    x, y = x.astype(np.float64), x.astype(np.float64).copy()
    c, s = cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
    a, b = (np.s_[..., 0:rot:2], np.s_[..., 1:rot:2]) if interleaved else (np.s_[..., :rot // 2], np.s_[..., rot // 2:rot])
    y[a] = x[a] * c - x[b] * s
    y[b] = x[b] * c + x[a] * s
    return y


def quantize4(x):
    """Codes [.., D / 2] and (scale, lowest) f16 [.., G, 2] of f32 x [.., D]."""
    D = x.shape[-1]
    G = D // 32
    g = np.clip(x.astype(F), F(-65504), F(65504)).reshape(x.shape[:-1] + (G, 32))
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        low = g.min(-1, keepdims=True).astype(np.float16)
        span = ((g.max(-1, keepdims=True) - low.astype(F)) * F(F(1) / F(15))).astype(F)
        scale = np.where(span < 0, F(0), span).astype(np.float16)
        q = np.clip(np.rint((g - low.astype(F)) / scale.astype(F)), 0, 15)
        c = np.where(scale > 0, q, 0)
    c = np.nan_to_num(c).astype(np.uint8).reshape(x.shape[:-1] + (G, 16, 2))
    byte = c[..., 0] | c[..., 1] << 4
    codes = np.swapaxes(byte, -1, -2).reshape(x.shape[:-1] + (D // 2,))
    return codes, np.concatenate([scale, low], -1)


def values4(codes, scales):
    """[.., D] in 64 bits of what codes and scales stand for."""
    G = scales.shape[-2]
    byte = np.swapaxes(codes.reshape(codes.shape[:-1] + (16, G)), -1, -2)
    c = np.stack([byte & 15, byte >> 4], -1).reshape(codes.shape[:-1] + (G, 32)).astype(np.float64)
    s = scales.astype(np.float64)
    return (c * s[..., :1] + s[..., 1:]).reshape(codes.shape[:-1] + (G * 32,))


def rows_of(pages, table, b):
    """[H, tokens, ..] of sequence b's pages [pages, H, size, ..]."""
    one = pages[[b]] if table is None else pages[table[b]]
    return np.concatenate(list(one), axis=1)


def attention(q, cache, past, table=None, counts=None, starts=None, scale=None, causal=True, window=0, half=False):
    """(y, sure): q [B, Hq, S, D]; rows behind a sequence's tokens are NaN.  sure:
    for each result the magnitudes its rounding errors are measured by, (largest
    sum |q khat| scale, largest |vhat|, largest code * scale of v, keys seen).
    half: khat and vhat are the nearest f16, +-65504 at most."""
    kc, ks, vc, vs = cache
    B, Hq, S, D = q.shape
    H = kc.shape[1]
    scale = 1 / np.sqrt(D) if scale is None else float(scale)
    y = np.full(q.shape, np.nan)
    sure = np.zeros(q.shape[:3] + (4,))
    for b in range(B):
        n = S if counts is None else int(counts[b])
        K, V = values4(rows_of(kc, table, b), rows_of(ks, table, b)), values4(rows_of(vc, table, b), rows_of(vs, table, b))
        if half:
            K, V = (np.clip(x, -65504, 65504).astype(np.float16).astype(np.float64) for x in (K, V))
        vsc = np.abs(rows_of(vs, table, b).astype(np.float64))
        for i in range(n):
            t = int(past[b]) + i
            end = min(K.shape[1], t + 1 if causal else int(past[b]) + n)
            first = max(0 if starts is None else int(starts[b]), t - window + 1 if window else 0, 0)
            for h in range(Hq):
                g = h * H // Hq
                if end <= first:
                    y[b, h, i] = 0
                    continue
                k, v = K[g, first:end], V[g, first:end]
                s = k @ q[b, h, i].astype(np.float64) * scale
                p = np.exp(s - s.max())
                y[b, h, i] = p @ v / p.sum()
                sure[b, h, i] = (np.abs(k * q[b, h, i].astype(np.float64)).sum(-1).max() * abs(scale), np.abs(v).max(),
                                 (vsc[g, first:end, :, 0] * 15 + vsc[g, first:end, :, 1]).max(), end - first)
    return y, sure
