"""What the losses hold in memory (CPU: the sizes that the library asks its caller for)."""
import pytest

from mlx_recurrence_amd import _lib

F32, BF16, F16 = 0, 1, 2
MIB = 1 << 20


def up(a, b):
    return (a + b - 1) // b * b


def sizes(rows, D, V, dtype, K=1):
    lib = _lib.load()
    return (lib.rr_linear_loss_workspace_bytes(rows, D, V, dtype, 0), lib.rr_linear_loss_workspace_bytes(rows, D, V, dtype, 1),
            *(lib.rr_linear_loss_state_bytes(rows, D, V, K, dtype, grad) for grad in (0, 1)))


SHAPES = [(T, D, V) for T in (1, 16, 40, 100, 256, 300, 756, 3000, 8192, 32768, 262144) for D in (64, 768, 2560, 7429, 16384, 65536)
          for V in (500, 5003, 32000, 65536, 141063, 262144) if T * D <= 1 << 31 and V * D <= 1 << 32]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_forward_workspace_holds_no_logits_beyond_256_mib(dtype):
    """A maximum and a sum per row and 256 words, and where the sums are made in parts at most 256 MiB of those."""
    for T, D, V in SHAPES:
        stats = up(V, 256) // 256 * up(T, 256) * 8
        assert sizes(T, D, V, dtype)[0] <= stats + 256 * MIB + 4096, (T, D, V)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_backward_workspace_holds_a_piece_of_the_gradient(dtype):
    """A piece of the logits' gradient: 512 MiB, or 2048 words of every row where those are more (two planes for up to 64
    rows of 16 bits).  Beside it fp32 sums of dhidden and, where dweight's are made in parts, of those: one copy, or
    parts of at most 256 MiB.  fp16: a copy of the hidden states."""
    size = 4 if dtype == F32 else 2
    for T, D, V in SHAPES:
        planes = 2 if dtype != F32 and T <= 64 else 1
        rows = 32 if T <= 32 else up(T, 256)
        piece = max(512 * MIB, 2048 * rows * size * planes)
        sums = max(rows * up(D, 256) * 4, 256 * MIB) + 256 * MIB
        copy = T * up(D, 64) * 2 if dtype == F16 else 0
        got = sizes(T, D, V, dtype)[1]
        assert got <= piece + sums + copy + rows * 16 + 4096, (T, D, V)
        if rows * up(V, 256) * size * planes > piece + sums + MIB:   # less than the whole gradient
            assert got - copy - rows * 16 < rows * up(V, 256) * size * planes, (T, D, V)


# rows, D, V, dtype, whether the logits are kept for the backward
@pytest.mark.parametrize("rows,D,V,dtype,kept", [
    (1, 5120, 131072, BF16, True), (16, 5120, 65536, BF16, True), (256, 64, 65536, F16, True),   # few rows
    (1536, 768, 32000, BF16, False), (1536, 768, 32000, F32, True), (8192, 2560, 65536, BF16, True),
    (32768, 2560, 131072, BF16, False), (8192, 4096, 131328, F16, False),   # more than 4 GiB
    (100_000, 64, 32000, F16, False), (8192, 64, 65536, F32, False), (777, 513, 10007, BF16, True),
])
def test_state_holds_the_logits_where_it_says(rows, D, V, dtype, kept):
    state = sizes(rows, D, V, dtype, K=4)[2:]
    size = 4 if dtype == F32 else 2
    logits = rows * up(V, 256) * 4
    assert state[1] - state[0] == (up(logits, 256) if kept else 0)
    copies = (rows + (V if D * size % 16 else 0)) * up(D, 64) * size
    assert state[0] <= copies + rows * (5 * 4 + 3 * 4 * 4) + 4096   # indices, lse, loss; four entries a row


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_state_without_room_for_the_logits(dtype):
    """grad = 2: the logits of up to 256 rows and of sums made in parts (128 MiB at most), no others."""
    lib = _lib.load()
    for T, D, V in SHAPES:
        without, small, full = (lib.rr_linear_loss_state_bytes(T, D, V, 1, dtype, grad) for grad in (0, 2, 1))
        logits = up(T * up(V, 256) * 4, 256)
        assert without <= small <= full and small - without in (0, logits)
        if T <= 256:
            assert small == full == without + logits
        else:
            assert small == without or logits <= 128 * MIB, (T, D, V)
    assert lib.rr_linear_loss_state_bytes(8, 8, 8, 1, dtype, 3) == 0 == lib.rr_linear_loss_state_bytes(8, 8, 8, 1, dtype, -1)


def test_backward_takes_a_state_of_either_size():
    """Refusals by the state's size (found before any work is enqueued: no pointer is read)."""
    lib, p = _lib.load(), 16
    for rows, D, V in ((8192, 2560, 65536), (4, 8, 10)):
        size = [lib.rr_linear_loss_state_bytes(rows, D, V, 1, 1, grad) for grad in (0, 1, 2)]
        run = lambda n: lib.rr_linear_loss_bwd(p, p, 1, rows, D, V, 1, 0.0, 1.0, 1, p, n, None, None, p, 1 << 40, None)  # noqa: E731,E501
        assert run(size[1]) == run(size[2]) == _lib.RR_OK
        assert run(size[2] - 1) == _lib.RR_EWORKSPACE


@pytest.mark.parametrize("rows,D,partial", [(1, 8, 1), (100, 1000, 13), (100, 1536, 13), (100, 1537, 50), (512, 2048, 256), (512, 2560, 256),
                                            (512, 2561, 256), (9000, 64, 512), (9000, 5120, 512), (3, 32768, 2)])
def test_layer_norm_backward_workspace(rows, D, partial):
    """Two partial rows (dweight's and dbias's) a workgroup, for two rows a wave or, where a workgroup takes a row, two
    rows a workgroup: the most that any input type's form needs (fp32 has a wave a row up to 1536 channels)."""
    assert _lib.load().rr_layer_norm_bwd_workspace_bytes(rows, D) == partial * 2 * D * 4
