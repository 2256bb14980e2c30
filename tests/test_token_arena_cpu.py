"""The work memory that a program of token steps asks for is what its launches touch: every lease
allocates and clears it. No device."""
import pytest

from synaptik_amd.native import validate_program_image
from synaptik_amd.program import ProgramBuilder

STATUS = 256  # the arena's first bytes


def rounded(n):
    return (n + 255) // 256 * 256


def norm_grad(R, C, gamma, beta):
    pb = ProgramBuilder()
    pb.layer_norm_grad(pb.input(R * C), pb.input(R * C), pb.output(R * C), R, C, gamma=pb.input(C),
                       dgamma=pb.output(C) if gamma else None, dbeta=pb.output(C) if beta else None)
    return validate_program_image(pb.image())


def embed_grad(N, V, D, accumulate=False):
    pb = ProgramBuilder()
    dw = pb.input(V * D, inout=True)
    pb.embed_grad(pb.input(max(1, N * D)), pb.input(max(1, N), "i32"), dw, N, V, D, accumulate=accumulate)
    return validate_program_image(pb.image())


def scan(B, T, D, back):
    pb = ProgramBuilder()
    n = B * T * D
    if back:
        pb.gated_scan_grad(*(pb.input(n) for _ in range(4)), pb.output(n), pb.output(n), B, T, D)
    else:
        pb.gated_scan(pb.input(n), pb.input(n), pb.output(n), B, T, D)
    return validate_program_image(pb.image())


@pytest.mark.parametrize("R,C", [(3, 7), (700, 300), (16384, 4096), (5, 20000)])
def test_layer_norm_grad_keeps_partial_sums_for_what_is_wanted(R, C):
    assert norm_grad(R, C, False, False) == STATUS
    both = norm_grad(R, C, True, True)
    assert both == norm_grad(R, C, True, False) == norm_grad(R, C, False, True)
    # a row of sums of either for each workgroup, of which there are at most R and 1024
    assert STATUS + 16 * C <= both <= STATUS + rounded(16 * C * min(R, 1024) + (16 * R if C > 16384 else 0))


@pytest.mark.parametrize("V,D", [(50, 9), (100000, 64), (1 << 21, 3)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embed_grad_of_few_rows_keeps_nothing(V, D, accumulate):
    for N in (0, 1, 255, 256):
        assert embed_grad(N, V, D, accumulate) == STATUS
    assert embed_grad(257, V, D, accumulate) > STATUS


@pytest.mark.parametrize("N,V,D", [(257, 70000, 3), (5000, 10007, 617), (8192, 40, 8)])
def test_embed_grad_of_a_sort_in_one_launch(N, V, D):
    """One list of keys and rows, parts of sums, a byte a table row where rows are cleared: nothing for
    counts, nor for a second list."""
    lists, parts = 8 * N + 32, 16 * D * ((N + 7) // 8) + 16
    assert embed_grad(N, V, D, True) <= STATUS + rounded(lists + parts)
    assert embed_grad(N, V, D) <= STATUS + rounded(lists + parts + V + 16)
    assert embed_grad(N, V, D, True) + (V - 256 if V < 1 << 20 else 0) <= embed_grad(N, V, D)


def test_embed_grad_of_tokens_of_one_digit():
    """Fewer than 512 table rows are sorted in one pass, from the tokens into one list."""
    N, D = 20000, 4
    assert embed_grad(N, 512, D) - embed_grad(N, 511, D) >= 8 * N - 512


@pytest.mark.parametrize("B,T,D", [(1, 65536, 512), (7, 1501, 617)])
def test_a_recurrence_keeps_its_own_direction_s_chunks(B, T, D):
    """A step of 16 bytes a chunk and channel and a copy of the states: fewer chunks back."""
    forward, back = scan(B, T, D, False), scan(B, T, D, True)
    assert STATUS < back < forward <= STATUS + rounded(4 * (4 * ((T + 127) // 128) + 1) * B * D)
    assert scan(B, 200, D, False) == scan(B, 200, D, True) == STATUS
