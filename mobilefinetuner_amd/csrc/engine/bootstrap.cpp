// libmft engine: the TCP sockets between the ranks of a job (see bootstrap.h).
#include "engine/bootstrap.h"

#include <arpa/inet.h>
#include <netdb.h>
#include <netinet/in.h>
#include <netinet/tcp.h>
#include <sys/socket.h>
#include <sys/time.h>
#include <unistd.h>

#include <algorithm>
#include <cerrno>
#include <chrono>
#include <cstdlib>
#include <cstring>
#include <stdexcept>
#include <thread>

namespace mft {
namespace eng {

int env_int(const char* k, int dflt) {
  const char* v = std::getenv(k);
  return v && *v ? std::atoi(v) : dflt;
}

double comm_timeout_s() { return (double)env_int("MFT_COMM_TIMEOUT", 600); }

bool send_all(int fd, const void* p, size_t n) {
  const char* c = static_cast<const char*>(p);
  while (n) {
    const ssize_t k = ::send(fd, c, n, MSG_NOSIGNAL);
    if (k <= 0) return false;
    c += k;
    n -= (size_t)k;
  }
  return true;
}

bool recv_all(int fd, void* p, size_t n) {
  char* c = static_cast<char*>(p);
  while (n) {
    const ssize_t k = ::recv(fd, c, n, 0);
    if (k <= 0) return false;
    c += k;
    n -= (size_t)k;
  }
  return true;
}

std::string resolve_ipv4(const std::string& host) {
  in_addr a{};
  if (::inet_pton(AF_INET, host.c_str(), &a) == 1) return host;
  addrinfo hints{}, *res = nullptr;
  hints.ai_family = AF_INET;
  hints.ai_socktype = SOCK_STREAM;
  const int rc = ::getaddrinfo(host.c_str(), nullptr, &hints, &res);
  if (rc != 0 || !res) throw std::runtime_error("comm: cannot resolve MASTER_ADDR '" + host + "': " + gai_strerror(rc));
  char buf[INET_ADDRSTRLEN] = {0};
  ::inet_ntop(AF_INET, &reinterpret_cast<sockaddr_in*>(res->ai_addr)->sin_addr, buf, sizeof(buf));
  ::freeaddrinfo(res);
  return buf;
}

namespace {

int comm_port() { return env_int("MFT_COMM_PORT", env_int("MASTER_PORT", 29500) + 1); }

sockaddr_in master_sockaddr() {
  const char* a = std::getenv("MASTER_ADDR");
  const std::string ip = resolve_ipv4(a && *a ? a : "127.0.0.1");
  sockaddr_in sa{};
  sa.sin_family = AF_INET;
  sa.sin_port = htons((uint16_t)comm_port());
  if (::inet_pton(AF_INET, ip.c_str(), &sa.sin_addr) != 1) throw std::runtime_error("comm: bad MASTER_ADDR " + ip);
  return sa;
}

void tune_socket(int fd) {
  int one = 1;
  ::setsockopt(fd, IPPROTO_TCP, TCP_NODELAY, &one, sizeof(one));
  timeval tv{};
  tv.tv_sec = (long)comm_timeout_s();
  ::setsockopt(fd, SOL_SOCKET, SO_RCVTIMEO, &tv, sizeof(tv));
}

}  // namespace

bool self_connected(int fd) {
  sockaddr_in a{}, b{};
  socklen_t na = sizeof(a), nb = sizeof(b);
  return ::getsockname(fd, reinterpret_cast<sockaddr*>(&a), &na) == 0 &&
         ::getpeername(fd, reinterpret_cast<sockaddr*>(&b), &nb) == 0 && a.sin_port == b.sin_port &&
         a.sin_addr.s_addr == b.sin_addr.s_addr;
}

// Star bootstrap: rank 0 listens and accepts world-1 connections (each peer sends magic + rank);
// the others connect (retrying while rank 0 comes up).  The port may lie in the range that the kernel hands out to
// connecting sockets: one of those can hold it when rank 0 comes to listen -- in use, or closed and in TIME_WAIT, which
// keeps a port from a listener unless both sockets have SO_REUSEADDR -- so the connecting ends set it as well, and rank 0
// tries again for a while (a peer's own attempts fail at once meanwhile, and are repeated).
std::vector<int> star_connect(int rank, int world) {
  sockaddr_in sa = master_sockaddr();
  std::vector<int> fds(world, -1);
  const int one = 1;
  const auto begin = std::chrono::steady_clock::now();
  auto past = [&](double s) { return std::chrono::duration<double>(std::chrono::steady_clock::now() - begin).count() > s; };
  if (rank == 0) {
    const double patience = std::min(comm_timeout_s(), 90.0);  // TIME_WAIT lasts a minute
    int lfd = -1;
    while (true) {
      lfd = ::socket(AF_INET, SOCK_STREAM, 0);
      ::setsockopt(lfd, SOL_SOCKET, SO_REUSEADDR, &one, sizeof(one));
      if (::bind(lfd, reinterpret_cast<sockaddr*>(&sa), sizeof(sa)) == 0 && ::listen(lfd, world) == 0) break;
      const int err = errno;
      ::close(lfd);
      if (err != EADDRINUSE || past(patience))
        throw std::runtime_error("comm: rank 0 cannot listen on port " + std::to_string(comm_port()) + ": " + std::strerror(err));
      std::this_thread::sleep_for(std::chrono::milliseconds(50));
    }
    for (int i = 1; i < world; ++i) {
      const int c = ::accept(lfd, nullptr, nullptr);
      uint32_t hdr[2] = {0, 0};
      if (c < 0 || !recv_all(c, hdr, sizeof(hdr)) || hdr[0] != kCommMagic || (int)hdr[1] <= 0 || (int)hdr[1] >= world ||
          fds[hdr[1]] >= 0) {
        ::close(lfd);
        throw std::runtime_error("comm: bad bootstrap connection");
      }
      tune_socket(c);
      fds[hdr[1]] = c;
    }
    ::close(lfd);
    return fds;
  }
  while (true) {
    const int fd = ::socket(AF_INET, SOCK_STREAM, 0);
    ::setsockopt(fd, SOL_SOCKET, SO_REUSEADDR, &one, sizeof(one));
    if (::connect(fd, reinterpret_cast<const sockaddr*>(&sa), sizeof(sa)) == 0 && !self_connected(fd)) {
      const uint32_t hdr[2] = {kCommMagic, (uint32_t)rank};
      if (!send_all(fd, hdr, sizeof(hdr))) {
        ::close(fd);
        throw std::runtime_error("comm: bootstrap send failed");
      }
      tune_socket(fd);
      fds[0] = fd;
      return fds;
    }
    ::close(fd);
    if (past(comm_timeout_s()))
      throw std::runtime_error("comm: timed out connecting to rank 0 on port " + std::to_string(comm_port()));
    std::this_thread::sleep_for(std::chrono::milliseconds(50));
  }
}

}  // namespace eng
}  // namespace mft
