"""The split of work between the warps of w4_vector_kernel
(hxinfer_b200/csrc/w4_linear.cu: launch_w4_vector_group, the kernel's head and
w4_fix_x), restated and checked on the CPU: every unit of x is put into fixed
point by exactly one warp, each warp reads only units that it or the warps it
meets at its barrier wrote, and every (tile, unit) is multiplied once.
Restates, and must track, the CUDA code."""
import pytest

MAX_WARPS, BARRIERS = 16, 16


def split(units, tiles, sms, ctas):
    """(ways, abreast) and the tiles of the largest and smallest CTA."""
    abreast = 2 if units < 4 * MAX_WARPS and tiles >= 6 * sms else 1
    ways = min(MAX_WARPS // abreast, units)
    counts = {tiles * (b + 1) // ctas - tiles * b // ctas for b in range(ctas)}
    return ways, abreast, counts


def converted(units, ways, abreast, warp):
    """Units that the warp converts: w4_fix_x from u0 + first on, every abreast-th."""
    way, first = warp % ways, warp // ways
    u0, u1 = units * way // ways, units * (way + 1) // ways
    mine = (u1 - u0 - first + abreast - 1) // abreast
    return [u0 + first + i * abreast for i in range(mine)], range(u0, u1)


@pytest.mark.parametrize("sms", [148, 132])
@pytest.mark.parametrize("units", list(range(1, 70)) + [127, 128, 320])
def test_one_writer_per_unit(units, sms):
    for tiles in (1, 2, sms - 1, sms, 6 * sms - 1, 6 * sms, 6 * sms + 5, 9504):
        for ctas in {min(tiles, sms), min(tiles, 3 * sms)}:
            ways, abreast, counts = split(units, tiles, sms, ctas)
            assert min(counts) >= 1
            writers = [0] * units
            for warp in range(ways * abreast):
                wrote, reads = converted(units, ways, abreast, warp)
                for u in wrote:
                    writers[u] += 1
                # the warps of a way meet at barrier 1 + way; a lone warp at none
                met = [converted(units, ways, abreast, w)[0] for w in range(warp % ways, ways * abreast, ways)]
                assert set(reads) <= {u for us in met for u in us}
            assert writers == [1] * units, (units, tiles, writers)
            assert abreast == 1 or 1 + ways <= BARRIERS
            for n in counts:  # tiles of a CTA: every one taken by one warp of each way
                taken = sorted(t for first in range(abreast) for t in range(first, n, abreast))
                assert taken == list(range(n))
