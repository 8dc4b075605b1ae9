"""The workspace of weighing, without a GPU: nothing is launched for it."""
import ctypes as C

import pytest


@pytest.mark.parametrize("quantized", [0, 1])
@pytest.mark.parametrize("heads, group, new, dim, page, pages", [(8, 8, 1, 128, 16, 8000), (2, 1, 8, 64, 48, 100), (4, 16, 1, 256, 128, 77), (8, 4, 3, 128, 64, 1)])
def test_scores_take_half_of_the_keys_at_most(heads, group, new, dim, page, pages, quantized):
    """Whatever a table has room for: beside them there are 8 bytes for each row of up to 256 parts of a sequence."""
    from nart_amd import hipq
    c = hipq.KvCacheStruct(k=1 << 20, v=1 << 20, k_scale=1 << 20 if quantized else None, v_scale=1 << 20 if quantized else None, pages=pages, heads=heads, page=page, dim=dim, type=2, quantized=quantized)

    def need(sequences, blocks, longest):
        d = hipq.KvWeighDesc(q=1 << 20, q_token=heads * group * dim, q_head=dim, starts=1 << 20, lens=1 << 20, blocks=1 << 20, weights=1 << 20, out=1 << 20, blocks_stride=blocks, sequences=sequences,
                             tokens=sequences * new, q_heads=heads * group, blocks_per_sequence=blocks, most_new=new, longest=longest, scale=0.1)
        got = hipq.lib().hipq_kv_weigh_workspace(C.byref(c), C.byref(d))
        assert got > 0, hipq.lib().hipq_last_error()
        return got
    rows, keys = new * group, pages * heads * page * dim * (1 if quantized else 2)
    for sequences in (1, 64):
        parts = sequences * heads * 256 * rows * 8 + 256
        for blocks in (1, pages, 1 << 13):
            assert need(sequences, blocks, 1 << 30) <= keys // 2 + parts
            assert need(sequences, blocks, 160) <= min(keys // 2, sequences * heads * rows * 160 * 4) + parts
