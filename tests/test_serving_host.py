"""Host-side checks of the serving operators that answer without a GPU."""
import pytest


def test_serving_operators_validation_without_gpu():
    """Argument checks of the serving entry points that run before any launch."""
    from smallaios_b200._lib import lib

    assert lib.sa_gqa_tree_attend(None, 0, None, None, None, 1, 1, 1, 8, 0, 0.0, None, 0, None) == 9
    assert lib.sa_kv_cache_keep_drafts(None, None, 1, 1, 1, None) == 9
    assert lib.sa_kv_block_means(None, 0, None, 0, 0, 1, None) == 9
    assert lib.sa_gqa_select_blocks(None, 0, None, 1, 1, 1, 8, None, 0, 0, 4, 1, 1, None, None) == 9
    assert lib.sa_gqa_sparse_attend(None, 0, None, None, 4, None, 1, 1, 1, 8, 0, 0.0, None, 0, None) == 9
    assert lib.sa_gqa_tree_workspace_bytes(None, 4, 1) == 0
    assert lib.sa_gqa_sparse_workspace_bytes(None, 4) == 0


def test_tree_layer_rows_must_match_batch_and_nodes():
    import torch

    import smallaios_b200 as sa

    with pytest.raises(ValueError):
        sa.tree_layer_step(torch.zeros(5, 8), None, None, None, 0, parents=torch.zeros(2, 3, dtype=torch.int32),
                           position_ids=None, cos_cache=None, sin_cache=None)
