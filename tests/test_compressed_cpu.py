"""What a compressed model does on the host before the device is touched."""
import numpy as np
import pytest
import scipy.sparse as sp

from recpack_amd.compressed import CompressedEASE, entries_by_row

X = sp.csr_matrix(np.array([[1, 0, 2], [0, 0, 0], [0, 3, 4], [5, 0, 0]]))


@pytest.mark.parametrize("kind", ["csr", "csc", "coo", "lil", "dok", "bsr"])
def test_entries_by_row_of_every_format(kind):
    indptr, indices = entries_by_row(X.asformat(kind), False)
    assert indptr.tolist() == [0, 2, 2, 4, 5]
    assert [sorted(indices[a:b].tolist()) for a, b in zip(indptr[:-1], indptr[1:])] == [[0, 2], [], [1, 2], [0]]


def test_repeated_entries_stay():
    coo = sp.coo_matrix((np.ones(4), ([2, 0, 2, 2], [1, 0, 1, 2])), shape=(3, 3))
    indptr, indices = entries_by_row(coo, False)
    assert indptr.tolist() == [0, 1, 1, 4] and indices.tolist() == [0, 1, 1, 2]


def test_room_behind_the_last_entry():
    room = X.copy()
    room.indices, room.data = np.append(room.indices, [9, 9]), np.append(room.data, [9, 9])
    assert entries_by_row(room, True)[1].tolist() == X.indices.tolist()


def test_weights_need_a_row_order():
    with pytest.raises(ValueError, match="CSR"):
        entries_by_row(X.tocsc(), True)


def test_scores_refuse_what_is_not_sparse():
    model = CompressedEASE()
    model.n_items_, model._rows, model._columns = 3, object(), None
    with pytest.raises(TypeError, match="sparse"):
        model.scores(X.toarray())
    with pytest.raises(ValueError, match="items"):
        model.scores(sp.csr_matrix((2, 5)))
