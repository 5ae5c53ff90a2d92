"""Results that overlap lists which blocks of the same launch go on reading are refused (no GPU needed)."""
import pytest

from test_attention_refusals import A, lib, refused  # noqa: F401  (lib: the fixture)
from test_tree_latent_refusals import commit_call, trees


@pytest.mark.parametrize("kw", [dict(path=5 * A), dict(path=5 * A + 4), dict(count=5 * A - 4), dict(nxt=5 * A + 4), dict(path=4 * A - 124), dict(count=4 * A + 124),
                                dict(nxt=4 * A + 64)])
def test_commits_over_sequences_and_tables(lib, kw):  # noqa: F811
    refused(lib, commit_call(lib, **kw), "overlap")


def test_commits_beside_them(lib):  # noqa: F811
    if lib.lag_hip_alloc(16):
        pytest.skip("a device is initialised in this process")
    for kw in (dict(path=5 * A + 8), dict(count=5 * A - 8), dict(nxt=4 * A + 128), dict(path=4 * A - 128), dict(path=5 * A, t=trees(seq_dev=None))):
        refused(lib, commit_call(lib, **kw), "not initialised")
