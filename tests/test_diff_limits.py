"""CPU: the largest numbers of rows that the Linear product with an activation
takes; more are refused on the host, before anything is launched."""
import ctypes as C

import rustnn_amd as R


def test_linear_rows():
    nb = C.c_size_t()
    code = lambda rows: R.lib().rnn_linear_act_workspace(rows, 1, 1, C.byref(nb))
    assert code((1 << 30) - 128) == R.RNN_OK
    assert code((1 << 30) - 127) == code(1 << 30) == R.RNN_E_UNSUPPORTED
