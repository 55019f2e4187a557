"""4-bit o_proj of a few tokens: whatever the number of clusters that are resident, the sums lie inside the shared memory that is asked for."""
import pytest

ROW = 20                    # floats between tokens of a tile's sums
LIMIT = 200 * 1024


@pytest.mark.parametrize("K", [64, 256, 2304, 4096, 4160, 8192, 8256, 11008, 14336, 16384, 16448, 28672, 32768])
@pytest.mark.parametrize("tokens", [1, 8, 9, 16])
def test_sums_fit(tokens, K, native_built):
    from helix_a2a_b200.ops._ext import ext
    nt = -(-tokens // 8)
    for hidden in list(range(16, 8193, 16)) + [1, 4096, 8192, 28672, 100000]:
        tiles = -(-hidden // 16)
        for resident in (1, 2, 3, 7, 16, 17, 18, 31, 33, 36, 37, 66, 73, 74, 148, 1000):
            cl, warps, columns, batch, batches, inboxes, size = ext().int4_few_plan(tokens, hidden, K, resident)
            assert cl in (1, 2, 4, 8) and 1 <= warps <= 16 and cl * warps * 256 >= K
            assert 1 <= columns <= min(tiles, resident) and batch >= 1
            # the walk of cluster 0, which has the most tiles: batch number `turn` leaves its sums in inbox turn % 2
            turns = -(-len(range(0, tiles, columns)) // batch)
            assert batches == turns
            used = 0 if cl == 1 else min(turns, 2)
            assert inboxes == used
            # floats: every warp's sums of a batch, then per inbox every rank's runs of four rows, 32 per tile and eight tokens
            assert 4 * (warps * batch * 8 * nt * ROW + used * cl * batch * 32 * nt * 4) <= size <= LIMIT
