"""How the ranks of a native job find each other (csrc/engine/bootstrap.cpp), in host processes: ports that something else
holds for a while, and a connection that a rank makes to itself."""
import os
import shutil
import socket
import subprocess
import time

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mobilefinetuner_amd", "csrc")

MAIN = r"""
#include <arpa/inet.h>
#include <netinet/in.h>
#include <sys/socket.h>
#include <unistd.h>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <exception>
#include "engine/bootstrap.h"
using namespace mft::eng;
static int port_of(int fd) {
  sockaddr_in a{};
  socklen_t n = sizeof(a);
  getsockname(fd, reinterpret_cast<sockaddr*>(&a), &n);
  return ntohs(a.sin_port);
}
int main(int argc, char** argv) {
  if (!strcmp(argv[1], "self")) {  // a socket connected to itself, and two ends of a pair
    sockaddr_in a{};
    a.sin_family = AF_INET, a.sin_addr.s_addr = htonl(INADDR_LOOPBACK);
    const int fd = socket(AF_INET, SOCK_STREAM, 0), l = socket(AF_INET, SOCK_STREAM, 0), c = socket(AF_INET, SOCK_STREAM, 0);
    if (bind(fd, (sockaddr*)&a, sizeof(a))) return 2;
    a.sin_port = htons(port_of(fd));
    if (connect(fd, (sockaddr*)&a, sizeof(a))) return 3;
    a.sin_port = 0;
    if (bind(l, (sockaddr*)&a, sizeof(a)) || listen(l, 1)) return 4;
    a.sin_port = htons(port_of(l));
    if (connect(c, (sockaddr*)&a, sizeof(a))) return 5;
    const int s = accept(l, nullptr, nullptr);
    printf("%d %d %d\n", self_connected(fd), self_connected(c), self_connected(s));
    return 0;
  }
  const int rank = atoi(argv[1]);
  try {
    const std::vector<int> fds = star_connect(rank, 2);
    const int fd = fds[rank ? 0 : 1];
    uint32_t w = 41;
    if (rank) {
      if (!send_all(fd, &w, 4) || !recv_all(fd, &w, 4)) return 6;
      printf("%u %d\n", w, port_of(fd));
    } else {
      if (!recv_all(fd, &w, 4)) return 7;
      ++w;
      char c;
      if (!send_all(fd, &w, 4) || recv_all(fd, &c, 1)) return 8;  // until the other end closes
      printf("%u\n", w);
    }
    close(fd);
  } catch (const std::exception& e) {
    printf("%s\n", e.what());
    return 1;
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def prog(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("bootstrap")
    (d / "main.cpp").write_text(MAIN)
    exe = str(d / "ranks")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, os.path.join(CSRC, "engine", "bootstrap.cpp"), str(d / "main.cpp"),
                    "-o", exe, "-lpthread"], check=True)
    return exe


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _start(prog, port):
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MFT_COMM_PORT=str(port), MFT_COMM_TIMEOUT="20")
    return [subprocess.Popen([prog, str(r)], stdout=subprocess.PIPE, text=True, env=env) for r in range(2)]


def _join(procs):
    out = [p.communicate(timeout=40)[0].split() for p in procs]
    assert [p.returncode for p in procs] == [0, 0] and out[0] == ["42"] and out[1][0] == "42", out
    return int(out[1][1])


def test_two_ranks(prog):
    _join(_start(prog, _free_port()))


def test_a_port_that_is_held_for_a_while(prog):
    """Rank 0 waits for it: its peers keep trying to connect for the same time."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        procs = _start(prog, s.getsockname()[1])
        time.sleep(1.5)
    _join(procs)


def test_the_port_of_an_earlier_connection(prog):
    """The connecting end of an earlier job leaves its port in TIME_WAIT for a minute; rank 0 of the next job can listen on it."""
    used = _join(_start(prog, _free_port()))
    t = time.time()
    _join(_start(prog, used))
    assert time.time() - t < 10


def test_a_socket_connected_to_itself_is_told_apart(prog):
    assert subprocess.run([prog, "self"], stdout=subprocess.PIPE, text=True, check=True).stdout.split() == ["1", "0", "0"]
