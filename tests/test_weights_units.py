"""lia_attention_weights counts units of work in 32 bits: the configurations it takes have fewer, leads and partly filled
blocks among them (on the CPU: a refused configuration has no workspace)."""
import pytest

BF16, FP4 = 2, 4


def _taken(lia, hq, hkv, keys, max_seqs, max_rows, page=4096):
    return lia.attention_weights_workspace_bytes(lia.AttentionConfig(
        hq, hkv, 64, page, 64, -(-keys // page), BF16, FP4, BF16, 0.125, max_seqs, max_rows, keys)) > 0


def _up(a, b):
    return -(-a // b)


def _units(hkv, group, keys, rows, seqs):
    """The largest count of either pass and form over a scan of `seqs` sequences of `rows` rows and `keys` keys each."""
    cols, p0 = rows * group, keys - rows
    few = hkv * seqs * _up(cols, 16) * _up(keys, 256)
    if rows < 16:
        return few
    stats = hkv * seqs * sum(_up(p0, 64) + _up(4 * (i + 1), group) + 3 for i in range(_up(cols, 256)))
    sums = 0
    for i in range(0, _up(keys, 512)) if keys < 1 << 20 else []:
        sums += _up(cols, 16) + 6 - max(0, 512 * i - p0) * group // 16
    if keys >= 1 << 20:  # (few rows: the blocks that skip units are the last one or two)
        sums = (_up(cols, 16) + 6) * (_up(keys, 512) - 2)
    return max(stats, hkv * seqs * sums)


@pytest.mark.parametrize("hkv,group,rows,seqs", [(8, 1, 16, 256), (8, 1, 17, 200), (1, 32, 16, 256), (64, 1, 16, 100),
                                                 (2, 8, 16, 64), (8, 4, 1, 256), (1, 1, 1, 1), (1, 1, 16, 1), (16, 1, 300, 16)])
def test_taken_configurations_count_in_32_bits(lia, hkv, group, rows, seqs):
    taken = refused = 0
    for bits in range(15 * 8, 32 * 8):
        keys = min(int(2 ** (bits / 8)), (1 << 32) - 1)
        if keys <= rows:
            continue
        if _taken(lia, hkv * group, hkv, keys, seqs, rows * seqs):
            taken += 1
            assert not refused
            assert _units(hkv, group, keys, rows, seqs) < 1 << 32 and (keys + 1024) * group < 1 << 32, keys
        else:
            refused += 1
            # and no configuration is refused that is far from the limit
            assert max(4 * _units(hkv, group, keys, rows, seqs), (keys + 1024) * group) >= 1 << 32, keys
    assert taken > 50 and (refused or hkv * group == 1)


def test_keys_near_the_last_32_bit_number(lia):
    """A step past the last key has to be counted too."""
    assert _taken(lia, 1, 1, (1 << 32) - 1025, 1, 1)
    assert not _taken(lia, 1, 1, (1 << 32) - 1024, 1, 1) and not _taken(lia, 1, 1, (1 << 32) - 1, 1, 1)


def test_many_sequences(lia):
    """A scan holds 256 of them: more than those do not add units, but slots and padding."""
    assert _taken(lia, 8, 8, 1 << 20, 1 << 16, 1 << 12)
    assert not _taken(lia, 8, 8, 1 << 10, 1 << 28, 1 << 12) and not _taken(lia, 8, 8, 1 << 10, (1 << 32) - 1, 1 << 12)
