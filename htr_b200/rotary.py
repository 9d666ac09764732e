"""Angles of a rotary embedding: cosines and sines of many positions, laid out once for `paged.rope_append`."""
import torch

from . import _lib


def angles(rows, dim, theta=1.0e6, first=0, factor=1.0, original=None, low=1.0, high=32.0, magnitude=1.0, device=torch.device("cuda")):
    """(cos, sin) float32 [rows, dim / 2] of the positions first ... first + rows - 1, for a rotary embedding of `dim` dimensions (even, at most 256).

    Pair i turns by theta^(-2 i / dim) a position.  For contexts longer than a model has learned, `factor` slows the pairs down: all of them, or where
    `original` (the positions that it learned) is given, those that turn at most `low` times within it by the whole factor, those that turn `high` times and more not at
    all, and between them by a share that lies linearly in their turns (not in the pair's index between two rounded borders, as some models have it: between the borders those have
    other frequencies).  Cosines and sines are multiplied by `magnitude` (it sharpens the scores by its
    square, as far as the rotated part of a head goes).

    Angles are taken in 64 bits.  A result is off by at most 7 * 2^-24 of magnitude, and by what the roundings of the frequency and the angle make, some 2^-51 of the angle.  Tables of many rows
    (64 a multiprocessor and more) are products of two angles' cosines and sines, in float32: the last bits of a position depend on which table it stands in."""
    both = _lib.host.rope_angles(rows, dim, theta, first, factor, original, low, high, magnitude, device)    # the usual case; None: whatever it does not take
    if both is not None:
        return both
    dev = torch.device(device)
    if dev.type != "cuda":
        raise _lib.HTRError("angles has no CPU path: device must be a CUDA device")
    if original is not None and not original > 0:
        raise _lib.HTRError(f"angles: original must be positive, got {original}")
    values = (float(theta), float(factor), 0.0 if original is None else float(original), float(low), float(high), float(magnitude))
    rows, dim, first = int(rows), int(dim), int(first)
    if rows < 0 or first < 0 or first + rows > 2 ** 31 - 1:
        raise _lib.HTRError(f"angles: positions must lie in [0, 2^31 - 1), got {rows} from {first}")
    if dim < 2 or dim % 2 or dim > 256:
        raise _lib.HTRError(f"angles: dim must be even and at most 256, got {dim}")
    dev = torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)
    cos, sin = (torch.empty((rows, dim // 2), dtype=torch.float32, device=dev) for _ in range(2))
    with torch.cuda.device(dev):
        rc = _lib.lib.htr_rope_angles(first, rows, dim, *values, cos.data_ptr(), sin.data_ptr(), torch.cuda.current_stream(dev).cuda_stream)
        _lib.check(rc, "htr_rope_angles")
    return cos, sin
