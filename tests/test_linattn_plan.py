"""CPU check of linear attention's workspace: what a call takes stays under its bound, whatever the heads are."""
import itertools

from linattn_plan import windows

BOUND = 1 << 30


def test_workspace_bound():
    calls = [(T, n, keys, heads, dk, dv, parts)
             for T, n in ((33, 1), (64, 1), (65, 1), (600, 1), (600, 9), (4096, 3), (8191, 200), (100000, 1), (1 << 20, 65536), (2 ** 31 - 1, 7))
             for keys, heads in ((1, 1), (16, 32), (32, 32), (256, 256), (1, 4096), (1024, 4096), (4096, 4096))
             for dk, dv in ((64, 16), (128, 128), (256, 256))
             for parts in (1, 2, 3)]
    for call, (rows, used, _) in zip(calls, windows(calls)):
        T = call[0]
        assert used <= BOUND, call
        assert rows % 64 == 0 and (rows == 0 or rows >= min(T, 128)), call


def test_workspace_of_ordinary_calls():
    """The engine's heads keep one window for prompts of thousands of rows; heads by the thousand have none."""
    (rows, _, _), = windows([(4096, 1, 16, 32, 128, 128, 3)])
    assert rows >= 4096
    (rows, _, _), = windows([(8192, 7, 16, 32, 128, 128, 1)])
    assert rows >= 8192
    (rows, used, _), = windows([(600, 1, 4096, 4096, 256, 256, 3)])
    assert rows == 0 and used == 0


def test_windows_of_long_calls():
    """As many rows as the bound leaves: half as many again would not fit."""
    for call in itertools.product((20000, 60000), (1, 40), (32, 256), (256,), (64, 256), (16,), (1, 3)):
        (rows, used, _), = windows([call])
        if 0 < rows < call[0]:
            assert used > BOUND // 4


def test_rows_token_by_token():
    """Where the chip is full, a sequence of a type with more bf16 parts goes token by token for longer: 48 rows of fp16
    take a quarter less time so at 128 channels, as many of bf16 a sixth more."""
    def brief(parts, n=64):
        return windows([(4096, n, 32, 32, 128, 128, parts)])[0][2]
    assert brief(3) >= 64 and 48 <= brief(2) < 64 and brief(1) < 48
    assert brief(3, n=1) == brief(2, n=1) == brief(1, n=1) == 32
