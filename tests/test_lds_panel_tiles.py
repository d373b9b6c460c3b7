"""CPU: the [32][64] panel tiles of the fused attention, whose swizzle sits in the source address of loads that go
straight to LDS: what a load puts into a slot is what the operand reads expect there, and the address identities that
let the kernels keep eight address registers hold for every lane."""
import lds_bank_model as m


def _slots():
    """LDS byte address of a 16-byte slot -> (row, piece) the four requests of a tile put there."""
    lib = m.index_lib()
    where = {}
    for chunk in range(4):
        for lane in range(64):
            where[16 * (64 * chunk + lane)] = (8 * chunk + lane // 8, lib.bsa_panel_src_piece(lane, chunk))
    return where


def test_requests_cover_whole_rows():
    where = _slots()
    assert sorted(where.values()) == [(r, p) for r in range(32) for p in range(8)]
    for chunk in range(4):                       # one request: 8 whole rows, each row's 8 lanes in one 128-byte line
        for lane in range(64):
            assert where[16 * (64 * chunk + lane)][0] == 8 * chunk + lane // 8


def test_row_operands_find_their_pieces():
    where = _slots()
    for step in range(4):
        for lane, a in enumerate(m.kernel_access("get_panel", arg0=step)):
            assert where[a] == (lane % 32, 2 * step + lane // 32)
            assert a == m.kernel_access("get_panel", arg0=0)[lane] ^ (32 * step)


def test_column_operands_find_their_pieces():
    where = _slots()
    base = m.kernel_access("get_panel_tr", arg0=0, arg1=0, arg2=0)
    for step in (0, 1):
        for half in (0, 1):
            for x0 in (0, 32):
                for lane, a in enumerate(m.kernel_access("get_panel_tr", arg0=step, arg1=half, arg2=x0)):
                    g, s = lane // 16, lane % 16
                    row = 16 * step + 8 * half + 4 * (g // 2) + s // 4
                    col = x0 + 16 * (g % 2) + 4 * (s % 4)
                    assert where[a - a % 16] == (row, col // 8) and a % 16 == 2 * (col % 8)
                    assert a == (base[lane] ^ (2 * x0) ^ (16 * half)) + 2048 * step + 1024 * half


def test_ordered_column_operands_find_their_columns():
    """A transposing read gives lane s of 16 the element s % 4 of what lanes s / 4, s / 4 + 4, + 8, + 12 address, one row each."""
    where, lib = _slots(), m.index_lib()
    for permuted, order in ((True, lib.bsa_perm16), (False, lib.bsa_swapped16)):
        for half in (0, 1):
            access = m.kernel_access("get_panel_tr_ordered", permuted=permuted, arg0=half)
            for lane in range(64):
                g, s = lane // 16, lane % 16
                for r in range(4):
                    a = access[16 * g + 4 * r + s // 4] + 2 * (s % 4)
                    row, piece = where[a - a % 16]
                    assert (row, 8 * piece + a % 16 // 2) == (8 * half + 4 * (g // 2) + r, order(lane % 32))


def test_swapped_rows_of_an_accumulator_are_an_operand():
    """Value v of lane half h is row 8 (v / 4) + 4 h + v % 4 of a product; with that row's index swapped, values 8 s .. 8 s + 7 are
    the contraction 16 s + 8 h + 0 .. 7 of a ds_read_b128 operand."""
    swapped = m.index_lib().bsa_swapped16
    assert sorted(swapped(i) for i in range(32)) == list(range(32))
    for h in (0, 1):
        for v in range(16):
            row = swapped(8 * (v // 4) + 4 * h + v % 4)
            assert row == 16 * (v // 8) + 8 * h + v % 8 == swapped(8 * (v // 4) + v % 4) + 8 * h
