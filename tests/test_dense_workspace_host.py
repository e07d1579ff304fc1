"""Dense attention's workspaces, without a GPU."""

import pytest

from test_train_ops_host import BWD, FWD, _call


@pytest.mark.parametrize("entry,args,change", [("svoo_dense_attention_fwd", FWD, dict(sq=1, sk=5000, ws_bytes=1 << 30)),
                                               ("svoo_dense_attention_bwd", BWD, dict(ws_bytes=1 << 30))])
@pytest.mark.parametrize("at", [0, 8, 4104])
def test_a_workspace_that_is_missing_or_at_an_odd_address(entry, args, change, at):
    rc, text = _call(entry, args, dict(change, ws=at or None))
    assert rc == -3 and "workspace" in text
