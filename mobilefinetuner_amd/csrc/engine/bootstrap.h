// libmft engine: the TCP sockets between the ranks of a job (no HIP): the communicator's bootstrap
// (comm.cpp: RCCL's unique id) and the wire of its loopback backend.
#pragma once
#include <cstddef>
#include <cstdint>
#include <string>
#include <vector>

namespace mft {
namespace eng {

constexpr uint32_t kCommMagic = 0x4D465443;  // "MFTC": guards against a stray listener on the port

int env_int(const char* k, int dflt);
double comm_timeout_s();  // MFT_COMM_TIMEOUT, default 600
bool send_all(int fd, const void* p, size_t n);
bool recv_all(int fd, void* p, size_t n);

// Star around rank 0, on MASTER_ADDR and MFT_COMM_PORT or MASTER_PORT + 1: rank 0 gets fds[r] for r >= 1,
// every other rank fds[0] = its connection to rank 0.
std::vector<int> star_connect(int rank, int world);

// The two ends of the connection are one socket: a TCP connect to a port of this host that nobody listens on
// succeeds when the kernel happens to pick that very port for the connecting socket.
bool self_connected(int fd);

// Resolve MASTER_ADDR (numeric IPv4 or a host name, getaddrinfo) to an IPv4 address string.
std::string resolve_ipv4(const std::string& host);

}  // namespace eng
}  // namespace mft
