"""CPU: a feed-forward block's workspace holds what its launches write there, from a restatement of how they cut their products."""
import itertools
import random

import pytest

SMS = 148                     # what the library counts without a device, and on a B200


def _up(a, b):
    return -(-a // b)


def _padded(n):
    return _up(n, 256) * 256


def _splits(tasks, stages, split):
    """Parts of k of products (rows, columns) over so many stages of 64: the least clocks over the column tiles and parts that a launch may take."""
    least_stages, per_column, least_clocks, start = (2, 12, 1500, 3000) if split else (4, 2, 200, 1500)
    best, least = 1, float("inf")
    for ct in (256, 192, 128, 64):
        tiles, values = sum(_up(m, 256) * _up(n, ct) for m, n in tasks), sum(m * _up(n, 32) * 32 for m, n in tasks)
        for s in range(1, 33):
            if s > 1 and stages // s < least_stages:
                break
            clocks = (5000 + values * s * 8 / 3400 if s > 1 else 0) + _up(tiles * s, SMS // 2) * (_up(stages, s) * max(per_column * ct, least_clocks) + start)
            if clocks < least:
                best, least = s, clocks
    return best


def _parts(tasks, stages, split):
    s = _splits(tasks, stages, split)
    return s * sum(m * _up(n, 32) * 32 * 4 for m, n in tasks) if s > 1 else 0


def _backward(dtype, M, C, F, O):
    """Bytes that a backward pass writes to: dg and du (float32: and the operands, in three parts each), the sums of the biases, then in one place the parts of dx (k: the hidden channels
    of dg, then those of du, each in whole stages), of the weights' gradients, and of the sums."""
    pitch, split = _up(F, 32) * 32, dtype == 0
    later = max(_parts([(M, C)], 2 * _up(F, 64), split), _parts([(F, C), (F, C), (O, F)], _up(M, 64), split), 512 * (2 * F + O if split else O) * 4)
    if not split:
        return _padded(4 * M * pitch) + _padded(_up(M, 256) * 8 * 2 * pitch * 4) + later
    cut = sum(_padded(6 * rows * _up(cols, 8) * 8) for rows, cols in ((M, C), (F, C), (F, C), (O, F), (M, O)))
    return cut + 2 * _padded(6 * M * pitch) + later


# Sizes whose hidden channels leave 1 to 32 in their last stage, so that twice them are an odd number of stages in one piece and an even one in two; and any sizes.
NAMED = [(885, 384, 1736, 384), (532, 768, 2080, 768), (233, 1280, 2968, 1280), (6457, 768, 4938, 768), (300, 64, 961, 64), (65, 384, 961, 384), (128, 64, 961, 8)]


@pytest.mark.parametrize("dtype", [0, 1])
def test_backward(dtype):
    from fovi_b200._lib import lib
    rng = random.Random(7)
    any_size = [tuple(int(2 ** rng.uniform(0, e)) for e in (15, 11, 12.5, 11)) for _ in range(1500)]
    last = [(m, c, 64 * f + rest, c) for m, c, f, rest in itertools.product((17, 65, 200, 513, 1100), (40, 384, 1280), (1, 9, 15, 27, 46, 80), (1, 32))]
    for sizes in NAMED + last + any_size:
        have, need = lib.fovi_gated_ffn_workspace_bytes(dtype, *sizes, 1), _backward(dtype, *sizes)
        assert have >= need, (sizes, have, need)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("tokens", [1, 7, 16])
def test_few_tokens_want_room_for_their_hidden_values_only(dtype, tokens):
    """Float32 hidden values, or two bf16 parts of each; the weights are read where they lie."""
    from fovi_b200._lib import lib
    for C, F, O in ((1280, 5120, 1280), (384, 1021, 384), (8, 40, 24)):
        assert lib.fovi_gated_ffn_workspace_bytes(dtype, tokens, C, F, O, 0) == tokens * _up(F, 32) * 32 * 4


@pytest.mark.parametrize("dtype", [0, 1])
def test_forward(dtype):
    """Of many tokens: h (float32: where it is not kept; and the operands, in three parts each), then the parts of the result."""
    from fovi_b200._lib import lib
    for M, C, F, O in NAMED + [(2000, 40, 65, 7), (4000, 384, 1021, 384), (16448, 1280, 5120, 1280), (5000, 1, 1, 1)]:
        if M <= 1024:
            continue
        parts, pitch = _parts([(M, O)], _up(F, 64), dtype == 0), _up(F, 32) * 32
        cut = sum(_padded(6 * rows * _up(cols, 8) * 8) for rows, cols in ((M, C), (F, C), (F, C), (O, F))) if dtype == 0 else 0
        for phase, h in ((0, _padded((6 if dtype == 0 else 2) * M * pitch)), (2, 0)):
            assert lib.fovi_gated_ffn_workspace_bytes(dtype, M, C, F, O, phase) >= cut + h + parts
