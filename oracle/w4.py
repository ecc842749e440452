"""Plain 4-bit linears in 64 bits: the definition in include/ornith_w4.h."""
import numpy as np


def codes_of(words):
    """uint32 [n, k/8] low-first words -> codes [n, k]."""
    words = np.asarray(words).view(np.uint32)
    return ((words[:, :, None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).reshape(words.shape[0], -1)


def weights(words, scales, zeros, group):
    """float64 [n, k]; scales float64 [n, groups], zeros [n, groups] or None."""
    c = codes_of(words).astype(np.float64)
    of = np.arange(c.shape[1]) // group
    z = 8.0 if zeros is None else np.asarray(zeros, np.float64)[:, of]
    return (c - z) * scales[:, of]


def packed(words, scales_bits32, zeros, group):
    """The banks of ornith_w4_pack: codes [n/16, k/128, 64, 4], meta [n/16, k/128, 16, 128/group]
    (group 256: [n/16, k/256, 16, 1])."""
    c = codes_of(words)
    n, k = c.shape
    tiles, blocks, groups = -(-n // 16), -(-k // 128), -(-k // group)
    full = np.full((tiles * 16, blocks * 128), 8, np.uint32)
    full[:n, :k] = c
    v = full.reshape(tiles, 16, blocks, 4, 4, 4, 2)                # tile, column, block, j, q, i, parity
    word = sum(v[..., i, e] << np.uint32(4 * i + 16 * e) for i in range(4) for e in range(2))
    codes = word.transpose(0, 2, 4, 1, 3).reshape(tiles, blocks, 64, 4)
    per = max(128 // group, 1)
    chunks = -(-blocks // 2) if group == 256 else blocks
    meta = np.full((tiles * 16, chunks * per), 8, np.uint32)
    z = np.uint32(8) if zeros is None else np.asarray(zeros, np.uint32)
    meta[:n, :groups] = (scales_bits32 & ~np.uint32(15)) | z
    return codes, meta.reshape(tiles, 16, chunks, per).transpose(0, 2, 1, 3)
